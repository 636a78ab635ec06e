// The KV-cache codec's entry points: checks, the kernels' parameters and their launch.
#include <algorithm>
#include <cstring>

#include "gpu_kv_codec_api.h"
#include "host_common.h"
#include "kv_codec.cuh"

namespace kv = confkv::kv;
using namespace confkv::host;

static_assert(LMCACHE_GPU_KV_INT8 == kv::kInt8 && LMCACHE_GPU_KV_FP8 == kv::kFp8 && LMCACHE_GPU_KV_MXFP4 == kv::kMxFp4);
static_assert(LMCACHE_GPU_KV_BF16 == kv::kBf16 && LMCACHE_GPU_KV_FP16 == kv::kFp16 && LMCACHE_GPU_KV_FP32 == kv::kFp32);

namespace {

constexpr uint64_t kMaxTiles = 1u << 30;   // of a launch

bool layout_ok(const lmcache_gpu_kv_layout* l)
{
    return l != nullptr && l->format >= kv::kInt8 && l->format <= kv::kMxFp4 && l->dtype >= kv::kBf16 &&
           l->dtype <= kv::kFp32 && l->planes >= 1 && l->planes <= 2 && l->layers >= 1 && l->layers <= 65535 &&
           l->heads >= 1 && l->heads <= 65535 && l->head_dim >= 1 && l->head_dim <= 65535;
}

// Vectors of an object; above kMaxVectors where it has too many.
uint64_t object_vectors(const lmcache_gpu_kv_layout& l, uint32_t tokens)
{
    const uint64_t rows = uint64_t{l.planes} * l.layers * l.heads;   // < 2^34
    return tokens != 0 && rows > kv::kMaxVectors / tokens ? uint64_t{kv::kMaxVectors} + 1 : rows * tokens;
}

bool aligned(const void* p, uint64_t to)
{
    return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

bool pages_ok(const lmcache_gpu_kv_layout& l, const lmcache_gpu_kv_pages& p)
{
    const uint32_t bases = l.planes * l.layers;
    if (p.bases == nullptr || bases > kv::kMaxBases || p.block_size == 0 || p.blocks > kv::kMaxVectors ||
        p.blocks * p.block_size > kv::kMaxVectors || p.block_stride < 0 || p.row_stride < 0 || p.head_stride < 0) {
        return false;
    }
    for (uint32_t k = 0; k < bases; ++k) {
        if ((p.bases[k] == nullptr && p.blocks != 0) || !aligned(p.bases[k], kv::element_bytes(l.dtype))) {
            return false;
        }
    }
    return true;
}

bool run_ok(const lmcache_gpu_kv_layout& l, const lmcache_gpu_kv_pages* pages, const lmcache_gpu_kv_run& r)
{
    if (r.count == 0) {
        return true;
    }
    const uint64_t vectors = object_vectors(l, r.tokens);
    if (vectors > kv::kMaxVectors) {
        return false;
    }
    const uint64_t size = kv::record_layout(l.format, l.head_dim, vectors).size;
    if (r.record == nullptr || !aligned(r.record, 16) || r.record_bytes < size || !aligned(r.ok, 4)) {
        return false;
    }
    if (r.count > 1 && (r.record_stride < 0 || static_cast<uint64_t>(r.record_stride) < size || r.record_stride % 16 != 0)) {
        return false;
    }
    if (vectors == 0) {
        return true;
    }
    if (pages != nullptr) {
        return r.slots != nullptr && aligned(r.slots, 8) && r.slots_stride >= 0;
    }
    return r.object != nullptr && aligned(r.object, kv::element_bytes(l.dtype)) && r.object_stride >= 0 &&
           r.plane_stride >= 0 && r.layer_stride >= 0 && r.token_stride >= 0 && r.head_stride >= 0;
}

using Kernel = void (*)(const kv::Args);

// How a launch cuts its work: 2^lg_group lanes share a vector.
struct Plan {
    Kernel kernel;
    uint32_t lg_group;
};

uint32_t log2_up(uint32_t n)
{
    uint32_t l = 0;
    while ((1u << l) < n) {
        ++l;
    }
    return l;
}

// The plan for vectors cut into granules of E values, in groups of at least 2^least lanes: of the R in the list the
// one that leaves the fewest lanes idle, the first of equals. No kernel: no group is large enough.
template <bool QUANTISE, int FMT, class T, int E, bool SPLIT, int SPAN, int... R>
Plan granule_plan(uint32_t head_dim, uint32_t least)
{
    const uint32_t granules = (head_dim + E - 1) / E;
    uint32_t most = 5;
    if (QUANTISE && FMT == kv::kMxFp4) {
        // the lanes that share a block
        least = std::max(least, log2_up(kv::kMxBlock / (E * SPAN)));
        most = SPAN > 1 ? least : most;
    }
    Plan best{nullptr, 0};
    uint32_t held = ~0u;
    (
        [&] {
            const uint32_t lg = std::max(log2_up((granules + R - 1) / R), least);
            if (lg <= most && (uint32_t{R} << lg) < held) {
                held = uint32_t{R} << lg;
                if constexpr (QUANTISE) {
                    best = Plan{kv::quantise_kernel<FMT, T, E, R, SPLIT, SPAN, -1>, lg};
                } else {
                    best = Plan{kv::dequantise_kernel<FMT, T, E, R, SPLIT, -1>, lg};
                }
            }
        }(),
        ...);
    return best;
}

// Granules of E values, R a lane in groups of 2^LG lanes, where a group holds the vector and no plan has been found
// before. Not for quantising MXFP4, whose groups are bound to its blocks.
template <bool QUANTISE, int FMT, class T, int E, bool SPLIT, int R, int LG>
void fit(uint32_t head_dim, Plan* p)
{
    if (p->kernel == nullptr && head_dim <= static_cast<uint32_t>((E * R) << LG)) {
        if constexpr (E == 1) {
            p->kernel = QUANTISE ? kv::quantise_single_kernel<FMT, T, R, LG> : kv::dequantise_single_kernel<FMT, T, R, LG>;
        } else if constexpr (QUANTISE) {
            p->kernel = kv::quantise_kernel<FMT, T, E, R, SPLIT, 1, LG>;
        } else {
            p->kernel = kv::dequantise_kernel<FMT, T, E, R, SPLIT, LG>;
        }
        p->lg_group = LG;
    }
}

template <bool QUANTISE, int FMT, class T, bool SPLIT>
Plan fit_pairs(uint32_t head_dim)
{
    Plan p{nullptr, 0};
    fit<QUANTISE, FMT, T, 2, SPLIT, 4, 2>(head_dim, &p);
    fit<QUANTISE, FMT, T, 2, SPLIT, 6, 2>(head_dim, &p);
    if constexpr (SPLIT) {
        fit<QUANTISE, FMT, T, 2, SPLIT, 4, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 6, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 4, 4>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 8, 4>(head_dim, &p);
    } else {
        fit<QUANTISE, FMT, T, 2, SPLIT, 8, 2>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 10, 2>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 6, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 8, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 12, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 2, SPLIT, 16, 3>(head_dim, &p);
    }
    fit<QUANTISE, FMT, T, 2, SPLIT, 16, 4>(head_dim, &p);
    fit<QUANTISE, FMT, T, 2, SPLIT, 16, 5>(head_dim, &p);
    return p;
}

// MXFP4 in granules of 2: a lane holds several granules of a block where the vector is short enough for it.
template <bool QUANTISE, class T, bool SPLIT>
Plan pair_plan(uint32_t head_dim)
{
    if constexpr (QUANTISE) {
        Plan p{nullptr, 0};
        if constexpr (SPLIT) {
            p = granule_plan<true, kv::kMxFp4, T, 2, SPLIT, 4, 8, 12, 16, 24>(head_dim, 2);
        } else {
            p = granule_plan<true, kv::kMxFp4, T, 2, SPLIT, 4, 8, 12, 16, 24, 32>(head_dim, 2);
        }
        return p.kernel != nullptr ? p : granule_plan<true, kv::kMxFp4, T, 2, SPLIT, 1, 8, 16>(head_dim, 0);
    } else {
        return fit_pairs<false, kv::kMxFp4, T, SPLIT>(head_dim);
    }
}

template <int FMT, class T>
Plan warp_plan(bool quantise)
{
    return Plan{quantise ? kv::quantise_warp_kernel<FMT, T> : kv::dequantise_warp_kernel<FMT, T>, 5};
}

// The largest granules that divide the vector and its addresses (`alignment`: a power of two that divides them all),
// and how many a lane holds. More a lane share the vector's address among more values, fewer keep the loads of
// neighbouring lanes together. Measured with 6 objects [2, 32, 256, 8, d] of bfloat16, us:
//   INT8 quantise   d = 200 (8): 8 a lane 89, 4 a lane 108; d = 72: 5 a lane 35, 3 a lane 46; d = 56: two lanes 29,
//                   one lane 33
//   INT8 dequantise d = 72 (8): 3 a lane 31, 5 a lane 37; d = 200: 4 a lane 75, 8 a lane 81
//   MXFP4 quantise  d = 40 (8): two granules of a block in a lane 19, one 29;  d = 100 (4): two 57, one 80;
//                   d = 66 (2): four 59, one 126
// With granules of 4 and fewer values instructions bound the kernel (419 of a warp for four vectors of 65 values, 52 a
// value, before `fit`), so the group is a constant and lane i's granules are at constant distances (INT8 quantise,
// known and not known when compiling: d = 100 (4) 49 and 61, d = 126 (2) 80 and 96), and single values are worked on in
// twos (d = 65: 67 and 92). R and LG are the fastest of 13 pairs each at 14 to 19 head sizes, of which a few:
//   d = 36 (4)  5 of two lanes 22, 3 of four 30       d = 204 (4)  8 of eight lanes 92, 16 of four 89 (252: 101, 110)
//   d = 34 (2)  6 of four 32, 4 of eight 54           d = 126 (2)  8 of eight 80, 16 of four 119, 4 of sixteen 112
//   d = 33 (1)  12 of four 34, 8 of eight 55          d = 127 (1)  8 of sixteen 113, 16 of eight 134
template <bool QUANTISE, int FMT, class T>
Plan granule_plan(uint32_t head_dim, uint64_t alignment)
{
    if (head_dim % 16 == 0 && alignment >= 32) {
        constexpr uint32_t least = FMT == kv::kMxFp4 ? 1 : 0;
        if constexpr (sizeof(T) == 4) {
            return granule_plan<QUANTISE, FMT, T, 16, false, 1, 2, 3, 1>(head_dim, least);
        } else {
            return granule_plan<QUANTISE, FMT, T, 16, false, 1, 4, 3, 5, 2, 1>(head_dim, least);
        }
    }
    if (head_dim % 8 == 0 && alignment >= 8 * sizeof(T)) {
        if constexpr (QUANTISE && FMT == kv::kMxFp4) {
            const Plan p = granule_plan<true, FMT, T, 8, false, 2, 4, 6, 8>(head_dim, 1);
            return p.kernel != nullptr ? p : granule_plan<true, FMT, T, 8, false, 1, 8, 6, 5>(head_dim, 1);
        } else if constexpr (QUANTISE) {
            return granule_plan<true, FMT, T, 8, false, 1, 8, 6, 5, 4, 3>(head_dim, 1);
        } else {
            return granule_plan<false, FMT, T, 8, false, 1, 4, 3>(head_dim, 1);
        }
    }
    if (head_dim % 4 == 0 && alignment >= 4 * sizeof(T)) {
        if constexpr (QUANTISE && FMT == kv::kMxFp4) {
            const Plan p = granule_plan<true, FMT, T, 4, false, 2, 4, 8, 16>(head_dim, 2);
            return p.kernel != nullptr ? p : granule_plan<true, FMT, T, 4, false, 1, 8, 16>(head_dim, 0);
        } else {
            Plan p{nullptr, 0};
            if constexpr (QUANTISE || sizeof(T) == 2) {
                fit<QUANTISE, FMT, T, 4, false, 5, 1>(head_dim, &p);
            }
            fit<QUANTISE, FMT, T, 4, false, 3, 2>(head_dim, &p);
            fit<QUANTISE, FMT, T, 4, false, 4, 2>(head_dim, &p);
            fit<QUANTISE, FMT, T, 4, false, 5, 2>(head_dim, &p);
            fit<QUANTISE, FMT, T, 4, false, 6, 2>(head_dim, &p);
            if constexpr (!QUANTISE && sizeof(T) == 4) {
                fit<QUANTISE, FMT, T, 4, false, 4, 3>(head_dim, &p);
            } else {
                fit<QUANTISE, FMT, T, 4, false, 8, 2>(head_dim, &p);
                fit<QUANTISE, FMT, T, 4, false, 12, 2>(head_dim, &p);
            }
            fit<QUANTISE, FMT, T, 4, false, 8, 3>(head_dim, &p);
            fit<QUANTISE, FMT, T, 4, false, 8, 4>(head_dim, &p);
            fit<QUANTISE, FMT, T, 4, false, 8, 5>(head_dim, &p);
            return p;
        }
    }
    const bool even = head_dim % 2 == 0 && alignment >= 2 * sizeof(T);
    if constexpr (FMT == kv::kMxFp4) {
        return even ? pair_plan<QUANTISE, T, false>(head_dim) : pair_plan<QUANTISE, T, true>(head_dim);
    } else {
        if (even) {
            return fit_pairs<QUANTISE, FMT, T, false>(head_dim);
        }
        Plan p{nullptr, 0};
        fit<QUANTISE, FMT, T, 1, false, 8, 2>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 12, 2>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 8, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 12, 3>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 8, 4>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 12, 4>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 16, 4>(head_dim, &p);
        fit<QUANTISE, FMT, T, 1, false, 16, 5>(head_dim, &p);
        return p;
    }
}

template <int FMT, class T>
Plan plan_of(uint32_t head_dim, uint64_t alignment, bool quantise)
{
    const Plan p = quantise ? granule_plan<true, FMT, T>(head_dim, alignment) : granule_plan<false, FMT, T>(head_dim, alignment);
    return p.kernel != nullptr ? p : warp_plan<FMT, T>(quantise);
}

template <int FMT>
Plan plan_of(const lmcache_gpu_kv_layout& l, uint64_t alignment, bool quantise)
{
    return l.dtype == kv::kBf16   ? plan_of<FMT, __nv_bfloat16>(l.head_dim, alignment, quantise)
           : l.dtype == kv::kFp16 ? plan_of<FMT, __half>(l.head_dim, alignment, quantise)
                                  : plan_of<FMT, float>(l.head_dim, alignment, quantise);
}

Plan plan_of(const lmcache_gpu_kv_layout& l, uint64_t alignment, bool quantise)
{
    return l.format == kv::kInt8  ? plan_of<kv::kInt8>(l, alignment, quantise)
           : l.format == kv::kFp8 ? plan_of<kv::kFp8>(l, alignment, quantise)
                                  : plan_of<kv::kMxFp4>(l, alignment, quantise);
}

// The largest power of two up to 32 that divides the addresses of all vectors: `bits` gathers the pointers and
// the strides in bytes of the dimensions that are longer than one.
uint64_t alignment_of(uint64_t bits)
{
    bits |= 32;
    return bits & (~bits + 1);
}

uint64_t strides_of_pages(const lmcache_gpu_kv_layout& l, const lmcache_gpu_kv_pages& p, int64_t element)
{
    uint64_t bits = 0;
    for (uint32_t k = 0; k < l.planes * l.layers; ++k) {
        bits |= reinterpret_cast<uintptr_t>(p.bases[k]);
    }
    bits |= p.blocks > 1 ? p.block_stride * element : 0;
    bits |= p.block_size > 1 ? p.row_stride * element : 0;
    bits |= l.heads > 1 ? p.head_stride * element : 0;
    return bits;
}

uint64_t strides_of_run(const lmcache_gpu_kv_layout& l, const lmcache_gpu_kv_run& r, int64_t element)
{
    uint64_t bits = reinterpret_cast<uintptr_t>(r.object);
    bits |= r.count > 1 ? r.object_stride * element : 0;
    bits |= l.planes > 1 ? r.plane_stride * element : 0;
    bits |= l.layers > 1 ? r.layer_stride * element : 0;
    bits |= r.tokens > 1 ? r.token_stride * element : 0;
    bits |= l.heads > 1 ? r.head_stride * element : 0;
    return bits;
}

int launch(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages, const lmcache_gpu_kv_run* runs,
           size_t count, int device, void* stream_ptr, bool quantise)
{
    if (!layout_ok(layout) || device < 0 || (runs == nullptr && count != 0)) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    const lmcache_gpu_kv_layout& l = *layout;
    if (pages != nullptr && !pages_ok(l, *pages)) {
        return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
    }
    for (size_t i = 0; i < count; ++i) {
        if (!run_ok(l, pages, runs[i])) {
            return LMCACHE_GPU_AESGCM_ERR_ARGUMENT;
        }
    }
    if (count == 0) {
        return LMCACHE_GPU_AESGCM_OK;
    }
    DeviceGuard guard(device);
    if (!guard.ok()) {
        return LMCACHE_GPU_AESGCM_ERR_CUDA;
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_ptr);
    const int64_t element = kv::element_bytes(l.dtype);

    kv::Args a;
    a.by_layers = kv::make_fast_div(l.layers);
    a.by_heads = kv::make_fast_div(l.heads);
    a.by_block = kv::make_fast_div(pages != nullptr ? pages->block_size : 1);
    a.head_dim = l.head_dim;
    a.layers = l.layers;
    a.paged = pages != nullptr ? 1 : 0;
    a.slots = 0;
    a.block_stride = a.row_stride = a.page_head_stride = 0;
    if (pages != nullptr) {
        a.slots = static_cast<uint32_t>(pages->blocks * pages->block_size);
        a.block_stride = pages->block_stride * element;
        a.row_stride = pages->row_stride * element;
        a.page_head_stride = pages->head_stride * element;
        std::memcpy(a.bases, pages->bases, sizeof(void*) * l.planes * l.layers);
    }
    const uint64_t page_bits = pages != nullptr ? strides_of_pages(l, *pages, element) : 0;
    Plan plan{};
    uint64_t tiles = 0;
    a.runs = 0;
    auto flush = [&]() -> cudaError_t {
        if (a.runs == 0) {
            return cudaSuccess;
        }
        const cudaError_t e = launch_pdl(plan.kernel, static_cast<uint32_t>(tiles), kv::kThreads, 0, s, a);
        a.runs = 0;
        tiles = 0;
        return e;
    };
    for (size_t i = 0; i < count; ++i) {
        const lmcache_gpu_kv_run& r = runs[i];
        const uint64_t vectors = object_vectors(l, r.tokens);
        const kv::RecordLayout rec = kv::record_layout(l.format, l.head_dim, vectors);
        const uint64_t alignment = alignment_of(pages != nullptr ? page_bits : strides_of_run(l, r, element));
        const Plan mine = plan_of(l, vectors == 0 ? 32 : alignment, quantise);
        const uint32_t units = vectors == 0 ? 1 : static_cast<uint32_t>(vectors);
        // as many objects at once as FastDiv can tell apart
        const uint32_t most = kv::kMaxVectors / units;
        for (uint32_t first = 0; first < r.count;) {
            const uint32_t n = r.count - first < most ? r.count - first : most;
            const uint64_t tile = kv::kThreads >> mine.lg_group;
            const uint64_t more = (uint64_t{n} * units + tile - 1) / tile;
            if (a.runs == kv::kMaxRuns ||
                (a.runs != 0 && (tiles + more > kMaxTiles || mine.kernel != plan.kernel))) {
                if (flush() != cudaSuccess) {
                    return LMCACHE_GPU_AESGCM_ERR_CUDA;
                }
            }
            plan = mine;
            a.lg_group = mine.lg_group;
            kv::Run& d = a.run[a.runs++];
            d.object = static_cast<char*>(r.object) + first * r.object_stride * element;
            d.object_stride = r.object_stride * element;
            d.plane_stride = r.plane_stride * element;
            d.layer_stride = r.layer_stride * element;
            d.token_stride = r.token_stride * element;
            d.head_stride = r.head_stride * element;
            d.slots = r.slots + first * r.slots_stride;
            d.slots_stride = r.slots_stride;
            d.record = static_cast<char*>(r.record) + first * r.record_stride;
            d.record_stride = r.record_stride;
            d.ok = r.ok != nullptr ? r.ok + first : nullptr;
            d.codes_end = rec.codes_end;
            d.scales_at = rec.scales_at;
            d.scales_end = rec.scales_end;
            d.record_bytes = rec.size;
            d.by_object = kv::make_fast_div(units);
            d.by_tokens = kv::make_fast_div(r.tokens == 0 ? 1 : r.tokens);
            d.units = n * units;
            d.empty = vectors == 0 ? 1 : 0;
            d.tile_start = static_cast<uint32_t>(tiles);
            d.header[0] = kv::kMagic;
            d.header[1] = r.tokens;
            d.header[2] = l.layers | l.heads << 16;
            d.header[3] = l.head_dim | static_cast<uint32_t>(l.format) << 16 | static_cast<uint32_t>(l.dtype) << 20 |
                          l.planes << 24;
            tiles += more;
            first += n;
        }
    }
    return cuda_rc(flush());
}

}  // namespace

extern "C" size_t lmcache_gpu_kv_record_size(const lmcache_gpu_kv_layout* layout, uint32_t tokens)
{
    if (!layout_ok(layout)) {
        return 0;
    }
    const uint64_t vectors = object_vectors(*layout, tokens);
    return vectors > kv::kMaxVectors ? 0 : kv::record_layout(layout->format, layout->head_dim, vectors).size;
}

extern "C" int lmcache_gpu_kv_quantise_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages,
                                             const lmcache_gpu_kv_run* runs, size_t count, int device, void* stream)
{
    return launch(layout, pages, runs, count, device, stream, true);
}

extern "C" int lmcache_gpu_kv_dequantise_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages,
                                               const lmcache_gpu_kv_run* runs, size_t count, int device, void* stream)
{
    return launch(layout, pages, runs, count, device, stream, false);
}
