// The entry points of a paged cache's requests: checks, the kernels' parameters and their launch.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "gpu_kv_paged_api.h"
#include "host_common.h"
#include "kv_attend.cuh"
#include "kv_paged.cuh"

namespace kv = confkv::kv;
using namespace confkv::host;

namespace {

bool aligned(const void* p, uint64_t to)
{
    return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

bool array_ok(const void* p, uint64_t to)
{
    return p != nullptr && aligned(p, to);
}

// The largest power of two up to 16 that divides all that `bits` gathers.
uint64_t alignment_of(uint64_t bits)
{
    bits |= 16;
    return bits & (~bits + 1);
}

// cudaLaunchKernelEx with programmatic stream serialization, as launch_pdl, for grids of two dimensions and without a key
// schedule's shared layout.
template <class A, class... More>
cudaError_t launch(void (*kernel)(A, More...), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t s, const A& a, More... more)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, more...);
}

// ------------------------------------------------------------------ block tables and slot maps

struct Range {
    uintptr_t begin, end;
};

Range range_of(const void* p, uint64_t bytes)
{
    const uintptr_t b = reinterpret_cast<uintptr_t>(p);
    return Range{b, p != nullptr ? b + bytes : b};
}

bool meet(const Range& a, const Range& b)
{
    return a.begin < a.end && b.begin < b.end && a.begin < b.end && b.begin < a.end;
}

// Whether any of n rows of `width` bytes, `stride` bytes apart, shares memory with a range; what lies between rows is not theirs.
bool rows_meet(const void* rows, uint64_t n, uint64_t stride, uint64_t width, const Range& r)
{
    const Range all = range_of(rows, n != 0 && width != 0 ? (n - 1) * stride + width : 0);
    if (!meet(all, r)) {
        return false;
    }
    if (n == 1 || r.begin <= all.begin) {
        return true;
    }
    const uint64_t row = (r.begin - all.begin) / stride, first = all.begin + row * stride;      // the last that begins at or before the range
    return r.begin < first + width || r.end > first + stride;
}

bool tables_ok(const lmcache_gpu_kv_tables& t)
{
    if (t.requests >= kv::kMaxRequests || t.width >= kv::kMost || t.ring >= kv::kMost || t.block_size == 0 ||
        uint64_t{t.blocks} * t.block_size > kv::kMost || t.block_size > kv::kMost || t.table_stride < 0) {
        return false;
    }
    if (!array_ok(t.cursor, 4) || !array_ok(t.cursor_after, 4) || (t.ring != 0 && !array_ok(t.free, 4)) ||
        !aligned(t.slots, 8) || !aligned(t.starts, 8) || (t.slots != nullptr && t.capacity >= kv::kMost) ||
        (t.slots == nullptr && t.starts != nullptr)) {
        return false;
    }
    const uint64_t n = t.requests;
    if (n != 0 && (!array_ok(t.held, 4) || !array_ok(t.lengths, 4) || !array_ok(t.kept, 4) ||
                   (t.width != 0 && !array_ok(t.tables, 4)) || (n > 1 && t.table_stride < t.width))) {
        return false;
    }
    if (t.table_stride > (int64_t{1} << 36)) {   // 2^24 rows of it stay below 2^63 bytes
        return false;
    }
    const Range out[] = {range_of(t.kept, 4 * n),
                         range_of(t.cursor_after, 8),
                         range_of(t.slots, 8 * t.capacity),
                         range_of(t.starts, 8 * (n + 1)),
                         range_of(t.free, 4 * uint64_t{t.ring})};
    const Range in[] = {range_of(t.held, 4 * n), range_of(t.lengths, 4 * n), range_of(t.cursor, 8)};
    const auto in_tables = [&](const Range& r) {
        return rows_meet(t.tables, n, 4 * static_cast<uint64_t>(t.table_stride), 4 * uint64_t{t.width}, r);
    };
    for (const Range& r : in) {
        if (in_tables(r)) {
            return false;
        }
    }
    for (size_t i = 0; i < std::size(out); ++i) {
        if (in_tables(out[i])) {
            return false;
        }
        for (size_t k = i + 1; k < std::size(out); ++k) {
            if (meet(out[i], out[k])) {
                return false;
            }
        }
        for (const Range& r : in) {
            if (meet(out[i], r)) {
                return false;
            }
        }
    }
    return true;
}

// ------------------------------------------------------------------ a layer of the cache

bool layer_ok(const lmcache_gpu_kv_layout* l, const lmcache_gpu_kv_pages* p, uint32_t layer)
{
    if (l == nullptr || p == nullptr || l->dtype < kv::kBf16 || l->dtype > kv::kFp32 || l->planes < 1 || l->planes > 2 ||
        l->layers < 1 || l->layers > 65535 || l->heads < 1 || l->heads > 65535 || l->head_dim < 1 || l->head_dim > 65535 ||
        layer >= l->layers) {
        return false;
    }
    if (p->bases == nullptr || p->block_size == 0 || p->blocks > kv::kMaxTokens ||
        p->blocks * p->block_size > kv::kMaxTokens || p->block_size > kv::kMaxTokens || p->block_stride < 0 || p->row_stride < 0 || p->head_stride < 0) {
        return false;
    }
    for (uint32_t plane = 0; plane < l->planes; ++plane) {
        const void* base = p->bases[plane * l->layers + layer];
        if ((base == nullptr && p->blocks != 0) || !aligned(base, kv::element_bytes(l->dtype))) {
            return false;
        }
    }
    return true;
}

// The bits of all addresses of the layer's vectors, in bytes.
uint64_t layer_bits(const lmcache_gpu_kv_layout& l, const lmcache_gpu_kv_pages& p, uint32_t layer, int64_t element)
{
    uint64_t bits = 0;
    for (uint32_t plane = 0; plane < l.planes; ++plane) {
        bits |= reinterpret_cast<uintptr_t>(p.bases[plane * l.layers + layer]);
    }
    bits |= p.blocks > 1 ? p.block_stride * element : 0;
    bits |= p.block_size > 1 ? p.row_stride * element : 0;
    bits |= l.heads > 1 ? p.head_stride * element : 0;
    return bits;
}

template <class G>
constexpr auto append_of = kv::append_kernel<G>;

// ------------------------------------------------------------------ attention

using AttendKernel = void (*)(const kv::AttendArgs);
using JoinKernel = void (*)(const kv::AttendArgs, uint32_t);

// How a launch does its work.
struct AttendPlan {
    AttendKernel kernel;
    JoinKernel join;
    uint32_t threads;
    uint32_t heads;             // query heads of a row
    uint32_t workers;
    kv::Cutting cutting;
    bool small;                 // copies of 4 or 8 bytes
    uint32_t shared;            // bytes of dynamic shared memory
    std::atomic<uint64_t>* allowed;     // devices on which the kernel may have them
};

constexpr uint32_t kSms = 148;
static_assert(4 * kSms <= kv::kMostWorkers);

template <class T, int VEC, int R, int GH, int U, int BLOCKS>
AttendPlan any_plan()
{
    return AttendPlan{kv::attend_any_kernel<T, VEC, R, GH, U, BLOCKS>, kv::join_kernel<T>, kv::kAttendThreads, GH, BLOCKS * kSms, kv::Cutting{2, 1}, false, 0, nullptr};
}

// Steps of four values (float32, and what is too long or too little aligned for the 16-bit kernels) or single ones; as many query heads in a row as
// registers hold, and no more than there are. Fewer blocks an SM than these spill less and hide less; measured, us: 17 requests of up to 3001 tokens, 3 key
// heads of 100 float32, 2 query heads each, 3 blocks 16.6, 4 blocks 18.2; 16 requests of up to 2048, 8 heads of 128, 8 query heads
// each, 2 blocks 46.1, 3 blocks 37.2, 4 blocks with half the tokens a turn 55.4; 32 requests of up to 4000 tokens, 16 query heads on a latent
// vector of 320 float32, four heads in a row 51, one 154; of 576, two in a row 91, one 165. In 16 bits, with queries at an odd element, on a latent
// vector of 320 four in a row 37, 52, 83 and 271 for 4, 8, 16 and 64 heads, one in a row 106, 189, 357 and 1329; of 576 two in a row 48 and 206 for 2 and 16, one 94
// and 475; 32 requests of up to 2048, 4 key heads of 320, 2 and 8 query heads each, 121 and 202, and 243 and 669; of 640, 2 each, 163 and 358.
template <class T>
AttendPlan any_plan(uint32_t d, uint32_t group, bool fours)
{
    if constexpr (sizeof(T) == 4) {
        if (fours && d <= 256) {
            return d <= 128   ? (group == 1   ? any_plan<T, 4, 4, 1, 8, 3>()
                                 : group == 2 ? any_plan<T, 4, 4, 2, 8, 3>()
                                 : group <= 4 ? any_plan<T, 4, 4, 4, 4, 4>()
                                              : any_plan<T, 4, 4, 8, 4, 3>())
                   : group == 1 ? any_plan<T, 4, 8, 1, 4, 3>()
                                : any_plan<T, 4, 8, 4, 4, 2>();
        }
    }
    if (fours && group > 1 && d > 256 && d <= 640) {
        return d <= 384 ? any_plan<T, 4, 12, 4, 2, 2>() : any_plan<T, 4, 20, 2, 2, 2>();
    }
    return d <= 128   ? (group == 1 ? any_plan<T, 1, 4, 1, 8, 3>() : any_plan<T, 1, 4, 8, 4, 3>())
           : d <= 256 ? (group == 1 ? any_plan<T, 1, 8, 1, 4, 3>() : any_plan<T, 1, 8, 4, 4, 2>())
           : fours    ? any_plan<T, 4, 32, 1, 2, 2>()
                      : any_plan<T, 1, 32, 1, 1, 2>();
}

template <class T, int DP, int NT, bool ONE, int STAGES, int BLOCKS, bool ALONE, bool SMALL>
AttendPlan mma_plan()
{
    static std::atomic<uint64_t> allowed{0};
    using Shape = kv::MmaShape<T, DP, NT, ONE, STAGES>;
    return AttendPlan{kv::attend_mma_kernel<T, DP, NT, ONE, STAGES, BLOCKS, ALONE, SMALL>, kv::join_kernel<T>, kv::kAttendThreads, Shape::kHeads, BLOCKS * kSms,
                      kv::Cutting{DP <= 128 ? 8u : 4u, 2}, SMALL, Shape::kShared, &allowed};
}

// `rows`: of all requests; with four a worker whole rows may go to a warp each.
template <class T, int DP, int NT, bool ONE, int STAGES, int BLOCKS>
AttendPlan mma_plan(uint64_t rows)
{
    return rows >= 4 * BLOCKS * kSms ? mma_plan<T, DP, NT, ONE, STAGES, BLOCKS, true, false>()
                                     : mma_plan<T, DP, NT, ONE, STAGES, BLOCKS, false, false>();
}

// Whether the 16-bit kernel takes vectors of this size, in a cache and of queries of this alignment.
bool mma_takes(const lmcache_gpu_kv_layout& l, uint64_t cache_alignment, uint64_t query_alignment)
{
    return l.dtype != kv::kFp32 && l.head_dim % 8 == 0 && l.head_dim <= (l.planes == 2 ? 256u : 576u) && cache_alignment >= 16 &&
           query_alignment >= 16;
}

template <class T, int DP, int NT, bool ONE, int STAGES, int BLOCKS>
AttendPlan wide_plan()
{
    static std::atomic<uint64_t> allowed{0};
    using Shape = kv::WideShape<T, DP, NT, ONE, STAGES>;
    return AttendPlan{kv::attend_wide_kernel<T, DP, NT, ONE, STAGES, BLOCKS>, kv::join_kernel<T>, kv::kWideThreads, Shape::kHeads,
                      BLOCKS * kSms, kv::Cutting{2, 1}, false, Shape::kShared, &allowed};
}

// Up to 8 query heads a key head, which fill a product's columns: warps of their own; more, or long vectors: warps that share a tile. Measured, us, own and
// shared: 32 requests of up to 4096 tokens, 8 key heads of 64 with 5, 8 and 16 query heads each 20.2 and 22.2, 19.7 and 23.2, 25 and 28 (so up to 16 there);
// of 128 with 5, 8 and 16 25.2 and 34.0, 26.3 and 34.6, 41 and 35; of 256 (up to 2048 tokens) with 5 and 8 30.2 and 39.7, 31.0 and 39.6; one latent vector of 128, 256
// and 320, 8 query heads, 64 requests of up to 8192 15.5 and 18.5, 23.1 and 26.5, 27.5 and 32.0; of 576, 16 query heads 134 and 44, 64 requests of up to 4096 with 128
// query heads 524 and 126. Stages and blocks: what fills shared memory.
template <class T>
AttendPlan mma_plan(const lmcache_gpu_kv_layout& l, uint32_t group, uint64_t requests)
{
    const uint32_t d = l.head_dim;
    const uint64_t rows = requests * l.heads;       // where a group is one row
    const bool many = group > 16;
    if (l.planes == 2) {
        if (group <= 8) {
            return d <= 64    ? mma_plan<T, 64, 1, false, 4, 3>(rows)
                   : d <= 128 ? mma_plan<T, 128, 1, false, 3, 2>(rows)
                   : d <= 192 ? mma_plan<T, 192, 1, false, 4, 1>(rows)
                              : mma_plan<T, 256, 1, false, 3, 1>(rows);
        }
        return d <= 64    ? (many ? wide_plan<T, 64, 2, false, 4, 2>() : mma_plan<T, 64, 2, false, 4, 2>(rows))
               : d <= 128 ? (many ? wide_plan<T, 128, 2, false, 3, 2>() : wide_plan<T, 128, 1, false, 3, 2>())
                          : (many ? wide_plan<T, 256, 2, false, 3, 1>() : wide_plan<T, 256, 1, false, 3, 1>());
    }
    if (group <= 8 && d <= 320) {
        return d <= 128   ? mma_plan<T, 128, 1, true, 5, 2>(rows)
               : d <= 256 ? mma_plan<T, 256, 1, true, 5, 1>(rows)
                          : mma_plan<T, 320, 1, true, 4, 1>(rows);
    }
    return d <= 128   ? (many ? wide_plan<T, 128, 2, true, 4, 2>() : wide_plan<T, 128, 1, true, 4, 2>())
           : d <= 256 ? (many ? wide_plan<T, 256, 2, true, 3, 1>() : wide_plan<T, 256, 1, true, 3, 1>())
           : d <= 320 ? (many ? wide_plan<T, 320, 2, true, 3, 1>() : wide_plan<T, 320, 1, true, 4, 1>())
                      : (many ? wide_plan<T, 576, 2, true, 2, 1>() : wide_plan<T, 576, 1, true, 2, 1>());
}

// Whether it takes them in copies of 4 or 8 bytes: even head sizes that are no multiple of 8, or addresses of less than 16 bytes. Measured, us, and in brackets with
// attend_any_kernel: 32 requests of up to 2048 tokens, 8 key heads of 36 with 4 query heads each 17 (53), of 64 with 1, 16 and 64 22 (29), 38 (98) and 112 (323),
// of 100 with 1, 4 and 64 29 (33), 26 (53) and 132 (341), of 130 and 250 with 4 64 (93) and 99 (101). 32 requests of up to 4000 tokens on a latent vector, all sizes in
// stages of 320 values: of 2, 36 and 100 with 4 heads 16 (23), 16 (22) and 19 (24), of 64 with 1, 4, 16 and 64 19 (15), 20 (22), 25 (28) and 70 (69), of 128 with 128 131 (125), of
// 300 with 1, 8 and 64 27 (38), 28 (50) and 110 (269).
bool mma_takes_small(const lmcache_gpu_kv_layout& l, uint64_t cache_alignment, uint64_t query_alignment)
{
    return l.dtype != kv::kFp32 && l.head_dim % 2 == 0 && l.head_dim <= (l.planes == 2 ? 256u : 320u) && cache_alignment >= 4 &&
           query_alignment >= 4;
}

template <class T>
AttendPlan small_plan(const lmcache_gpu_kv_layout& l)
{
    const uint32_t d = l.head_dim;
    if (l.planes == 1) {
        return mma_plan<T, 320, 1, true, 4, 1, false, true>();
    }
    return d <= 64    ? mma_plan<T, 64, 1, false, 4, 3, false, true>()
           : d <= 128 ? mma_plan<T, 128, 1, false, 3, 2, false, true>()
                      : mma_plan<T, 256, 1, false, 3, 1, false, true>();
}

AttendPlan attend_plan(const lmcache_gpu_kv_layout& l, uint32_t group, uint64_t cache_alignment, uint64_t query_alignment,
                       uint64_t requests)
{
    if (mma_takes(l, cache_alignment, query_alignment)) {
        return l.dtype == kv::kBf16 ? mma_plan<__nv_bfloat16>(l, group, requests) : mma_plan<__half>(l, group, requests);
    }
    if (mma_takes_small(l, cache_alignment, query_alignment)) {
        return l.dtype == kv::kBf16 ? small_plan<__nv_bfloat16>(l) : small_plan<__half>(l);
    }
    const bool fours = l.head_dim % 4 == 0 && cache_alignment >= 4 * kv::element_bytes(l.dtype);
    return l.dtype == kv::kBf16   ? any_plan<__nv_bfloat16>(l.head_dim, group, fours)
           : l.dtype == kv::kFp16 ? any_plan<__half>(l.head_dim, group, fours)
                                  : any_plan<float>(l.head_dim, group, fours);
}

// Once for each device and kernel: more shared memory than 48 KiB has to be asked for.
cudaError_t allow_shared(const AttendPlan& p, int device)
{
    const uint64_t bit = device < 64 ? uint64_t{1} << device : 0;
    if (p.allowed == nullptr || (p.allowed->load(std::memory_order_acquire) & bit) != 0) {
        return cudaSuccess;
    }
    const cudaError_t e = cudaFuncSetAttribute(p.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(p.shared));
    if (e == cudaSuccess) {
        p.allowed->fetch_or(bit, std::memory_order_release);
    }
    return e;
}

// The parts of the workspace, in bytes behind its start.
struct Workspace {
    uint64_t sums, partial, size;
};

Workspace workspace_of(const AttendPlan& p, uint32_t value_dim)
{
    Workspace w{};
    const uint64_t places = uint64_t{2} * p.workers * p.heads;
    w.sums = uint64_t{p.workers} * sizeof(int4);
    w.partial = w.sums + places * sizeof(float2);
    w.size = w.partial + places * ((value_dim + 3) / 4 * 4) * sizeof(float);
    return w;
}

bool heads_ok(const lmcache_gpu_kv_layout& l, uint32_t query_heads, uint32_t value_dim)
{
    return l.heads >= 1 && l.heads <= 65535 && query_heads >= 1 && query_heads <= 65535 && query_heads % l.heads == 0 &&
           l.head_dim >= 1 && l.head_dim <= 1024 && value_dim >= 1 && value_dim <= l.head_dim && l.planes >= 1 &&
           l.planes <= 2 && (l.planes == 1 || value_dim == l.head_dim) && l.dtype >= kv::kBf16 && l.dtype <= kv::kFp32;
}

}  // namespace

extern "C" int lmcache_gpu_kv_resize_async(const lmcache_gpu_kv_tables* tables, int device, void* stream)
{
    if (tables == nullptr || device < 0 || !tables_ok(*tables)) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    const lmcache_gpu_kv_tables& t = *tables;
    DeviceGuard guard(device);
    if (!guard.ok()) {
        return LMCACHE_GPU_AESGCM_ERR_CUDA;
    }
    kv::ResizeArgs a{};
    a.tables = t.tables;
    a.table_stride = t.table_stride;
    a.held = t.held;
    a.lengths = t.lengths;
    a.free = t.free;
    a.cursor = t.cursor;
    a.kept = t.kept;
    a.cursor_after = t.cursor_after;
    a.slots = t.slots;
    a.starts = t.starts;
    a.capacity = t.slots != nullptr ? static_cast<uint32_t>(t.capacity) : kv::kMost;
    a.requests = t.requests;
    a.limit = kv::row_limit(t.width, t.block_size);
    a.blocks = t.blocks;
    a.ring = t.ring;
    // a thread a request or two: a token each for 256, 512 and 1024 requests takes 3.2, 3.9 and 5.5 us with 256 threads and 4.3, 4.7 and 5.6 with 1024,
    // 100 tokens each 3.6, 4.1 and 6.3 and 4.7, 5.2 and 5.4
    const uint32_t threads = t.requests <= 512 ? 256 : 1024;
    a.per = (t.requests + threads - 1) / threads;
    a.by_block = kv::make_fast_div(t.block_size);
    // the slots, and a few names a request
    const uint64_t units = std::max<uint64_t>(t.slots != nullptr ? t.capacity : 0, uint64_t{t.requests} * std::min(t.width, 32u));
    const uint64_t grid = std::clamp<uint64_t>((units + threads - 1) / threads, 1, kSms);
    return cuda_rc(launch(threads == 256 ? kv::resize_kernel<256> : kv::resize_kernel<1024>, dim3(static_cast<uint32_t>(grid)), threads, 0,
                          reinterpret_cast<cudaStream_t>(stream), a));
}

extern "C" int lmcache_gpu_kv_append_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages, uint32_t layer,
                                           const lmcache_gpu_kv_vectors* vectors, int device, void* stream)
{
    if (!layer_ok(layout, pages, layer) || vectors == nullptr || device < 0) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    const lmcache_gpu_kv_layout& l = *layout;
    const lmcache_gpu_kv_vectors& v = *vectors;
    const int64_t element = kv::element_bytes(l.dtype);
    const bool two = l.planes == 2;
    if (uint64_t{l.heads} * l.head_dim > (1u << 30) || v.tokens > kv::kMaxTokens || v.key_stride < 0 || v.key_head_stride < 0 ||
        (two && (v.value_stride < 0 || v.value_head_stride < 0))) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    if (v.tokens == 0) {
        return LMCACHE_GPU_AESGCM_OK;
    }
    if (!array_ok(v.keys, element) || (two && !array_ok(v.values, element)) || !array_ok(v.slots, 8)) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    if (pages->blocks == 0) {
        return LMCACHE_GPU_AESGCM_OK;
    }
    DeviceGuard guard(device);
    if (!guard.ok()) {
        return LMCACHE_GPU_AESGCM_ERR_CUDA;
    }
    kv::AppendArgs a{};
    uint64_t bits = layer_bits(l, *pages, layer, element) | l.head_dim * element;
    for (uint32_t p = 0; p < l.planes; ++p) {
        a.source[p] = static_cast<const char*>(p == 0 ? v.keys : v.values);
        a.token_stride[p] = (p == 0 ? v.key_stride : v.value_stride) * element;
        a.head_stride[p] = (p == 0 ? v.key_head_stride : v.value_head_stride) * element;
        a.plane[p] = static_cast<char*>(pages->bases[p * l.layers + layer]);
        bits |= reinterpret_cast<uintptr_t>(a.source[p]);
        bits |= v.tokens > 1 ? a.token_stride[p] : 0;
        bits |= l.heads > 1 ? a.head_stride[p] : 0;
    }
    a.block_stride = pages->block_stride * element;
    a.row_stride = pages->row_stride * element;
    a.page_head_stride = pages->head_stride * element;
    a.cache_slots = static_cast<uint32_t>(pages->blocks * pages->block_size);
    const uint32_t size = static_cast<uint32_t>(alignment_of(bits));
    a.by_vector = kv::make_fast_div(static_cast<uint32_t>(l.head_dim * element / size));
    a.by_heads = kv::make_fast_div(l.heads);
    a.by_block = kv::make_fast_div(pages->block_size);
    const uint64_t per_token = uint64_t{l.heads} * a.by_vector.d;
    const uint64_t most = std::max<uint64_t>(1, (uint64_t{1} << 30) / per_token);
    const auto kernel = size == 16 ? append_of<uint4> : size == 8 ? append_of<uint2> : size == 4 ? append_of<uint32_t> : append_of<uint16_t>;
    for (uint64_t first = 0; first < v.tokens; first += most) {
        const uint64_t n = std::min(most, v.tokens - first);
        kv::AppendArgs b = a;
        b.slots = v.slots + first;
        for (uint32_t p = 0; p < l.planes; ++p) {
            b.source[p] += first * a.token_stride[p];
        }
        b.units = static_cast<uint32_t>(n * per_token);
        const uint32_t per_block = kv::kAppendThreads * kv::kAppendUnits;
        const cudaError_t e = launch(kernel, dim3((b.units + per_block - 1) / per_block, l.planes), kv::kAppendThreads, 0,
                                     reinterpret_cast<cudaStream_t>(stream), b);
        if (e != cudaSuccess) {
            return LMCACHE_GPU_AESGCM_ERR_CUDA;
        }
    }
    return LMCACHE_GPU_AESGCM_OK;
}

extern "C" size_t lmcache_gpu_kv_attend_workspace_size(const lmcache_gpu_kv_layout* layout, uint32_t query_heads, uint32_t value_dim)
{
    if (layout == nullptr || !heads_ok(*layout, query_heads, value_dim)) {
        return 0;
    }
    // the most that the kernel of any alignment takes; the cache's and the query's need not be the same
    const uint32_t group = query_heads / layout->heads;
    const uint64_t element = kv::element_bytes(layout->dtype);
    uint64_t most = 0;
    for (uint64_t cache = element; cache <= 16; cache *= 2) {
        for (uint64_t query = element; query <= 16; query *= 2) {
            most = std::max(most, workspace_of(attend_plan(*layout, group, cache, query, 0), value_dim).size);
        }
    }
    return most;
}

extern "C" int lmcache_gpu_kv_attend_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages, uint32_t layer,
                                           const lmcache_gpu_kv_attention* attention, int device, void* stream)
{
    if (!layer_ok(layout, pages, layer) || attention == nullptr || device < 0) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    const lmcache_gpu_kv_layout& l = *layout;
    const lmcache_gpu_kv_attention& t = *attention;
    const int64_t element = kv::element_bytes(l.dtype);
    if (!heads_ok(l, t.query_heads, t.value_dim) || t.requests >= kv::kMaxRequests || t.width >= kv::kMost ||
        t.query_stride < 0 || t.query_head_stride < 0 || t.out_stride < 0 || t.out_head_stride < 0 || t.lse_stride < 0 ||
        t.table_stride < 0 || !std::isfinite(t.scale * kv::kLog2e)) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    const uint64_t query_bits = reinterpret_cast<uintptr_t>(t.query) | (t.requests > 1 ? t.query_stride * element : 0) |
                                (t.query_heads > 1 ? t.query_head_stride * element : 0);
    const uint64_t cache_alignment = alignment_of(layer_bits(l, *pages, layer, element));
    const AttendPlan plan = attend_plan(l, t.query_heads / l.heads, cache_alignment, alignment_of(query_bits), t.requests);
    const Workspace w = workspace_of(plan, t.value_dim);
    if (!array_ok(t.workspace, 16) ||
        t.workspace_bytes < std::max<uint64_t>(w.size, lmcache_gpu_kv_attend_workspace_size(layout, t.query_heads, t.value_dim))) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    if (t.requests == 0) {
        return LMCACHE_GPU_AESGCM_OK;
    }
    if (!array_ok(t.query, element) || !array_ok(t.out, element) || !aligned(t.lse, 4) || !array_ok(t.lengths, 4) ||
        (t.width != 0 && !array_ok(t.tables, 4))) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    kv::AttendArgs a{};
    a.group = t.query_heads / l.heads;
    a.chunks = (a.group + plan.heads - 1) / plan.heads;
    a.rows = l.heads * a.chunks;
    a.limit = kv::row_limit(t.width, pages->block_size);
    // the units of all requests, a row of each, are counted in 32 bits
    if (uint64_t{t.requests} * (a.limit / kv::kTile + 1 + kv::kRowUnits) >= (uint64_t{1} << 31)) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    DeviceGuard guard(device);
    if (!guard.ok()) {
        return LMCACHE_GPU_AESGCM_ERR_CUDA;
    }
    a.planes[0] = static_cast<const char*>(pages->bases[layer]);
    a.planes[1] = static_cast<const char*>(pages->bases[(l.planes - 1) * l.layers + layer]);
    if (pages->blocks == 0) {
        a.planes[0] = a.planes[1] = static_cast<const char*>(t.workspace);      // never read, but an address
    }
    a.block_stride = pages->block_stride * element;
    a.row_stride = pages->row_stride * element;
    a.page_head_stride = pages->head_stride * element;
    a.query = static_cast<const char*>(t.query);
    a.query_stride = t.query_stride * element;
    a.query_head_stride = t.query_head_stride * element;
    a.out = static_cast<char*>(t.out);
    a.out_stride = t.out_stride * element;
    a.out_head_stride = t.out_head_stride * element;
    a.lse = t.lse;
    a.lse_stride = t.lse_stride;
    a.tables = t.tables;
    a.table_stride = t.table_stride;
    a.lengths = t.lengths;
    char* const space = static_cast<char*>(t.workspace);
    a.cut = reinterpret_cast<int4*>(space);
    a.partial_sums = reinterpret_cast<float2*>(space + w.sums);
    a.partial = reinterpret_cast<float*>(space + w.partial);
    a.requests = t.requests;
    a.blocks = static_cast<uint32_t>(pages->blocks);
    a.window = t.window;
    a.head_dim = l.head_dim;
    a.value_dim = t.value_dim;
    a.value_pad = (t.value_dim + 3) / 4 * 4;
    a.scale = t.scale * kv::kLog2e;
    a.by_block = kv::make_fast_div(pages->block_size);
    a.by_chunks = kv::make_fast_div(a.chunks);
    a.cutting = plan.cutting;
    a.workers = plan.workers;
    a.cut_by_row = uint64_t{t.requests} * a.rows * std::min(plan.heads, a.group) <= kSms ? 1 : 0;
    a.granule = !plan.small ? 16 : std::min(cache_alignment, alignment_of(l.head_dim * element)) >= 8 ? 8 : 4;
    a.by_vector = kv::make_fast_div(std::max(1u, static_cast<uint32_t>(l.head_dim * element / a.granule)));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = allow_shared(plan, device);
    if (e != cudaSuccess) {
        return LMCACHE_GPU_AESGCM_ERR_CUDA;
    }
    e = launch(plan.kernel, dim3(plan.workers), plan.threads, plan.shared, s, a);
    // rows that no length makes long enough to be cut need no joining
    const uint32_t most = t.window != 0 ? std::min(t.window, a.limit) : a.limit;
    if (e == cudaSuccess && kv::tiles_of(kv::Span{0, most}, kv::kTile) > plan.cutting.whole_tiles) {
        // few rows have many pieces each: their values are shared out among as many blocks as there are SMs, one row's among those of
        // a worker's place where rows are many (one request, one key head, 131072 tokens: 27.9 us, and 42.0 the other way; 128 requests
        // of one key head: 19.6, and 21.3 with blocks that look at a row each)
        const uint32_t heads = std::min(plan.heads, a.group), rows = a.cut_by_row != 0 ? t.requests * a.rows : plan.workers;
        const uint32_t shares = a.cut_by_row != 0 ? std::clamp(kSms / (rows * heads), 1u, (a.value_pad + 15) / 16) : 1u;
        e = launch(plan.join, dim3(rows, heads, shares), kv::kAttendThreads, 0, s, a, plan.heads);
    }
    return cuda_rc(e);
}
