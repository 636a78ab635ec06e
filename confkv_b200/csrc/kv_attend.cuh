// Attention of one new token a request over a paged cache (include/gpu_kv_paged_api.h).
//
// For a query head q and the tokens i of its request s_i = scale q k_i, out = sum_i e^(s_i - m) v_i / l with m = max s_i and l = sum
// e^(s_i - m); any split of the tokens gives pieces (m, l, sum e^(s_i - m) v_i) that are joined by weights e^(m - max m), so one pass
// over the cache is enough, in any order. Exponents are taken to base 2, the scale times log2 e.
//
// A token of a key head is 4 d bytes (16 bits, keys and values) for 4 d operations a query head: with 8 query heads 8 operations a
// byte, where the copy rate of 6.55 TB/s and 1670 TFLOP/s meet at 255. So memory bounds the kernels, each byte is read once, and the
// matrix instructions that one warp issues alone (16 x 8 x 16, 2 cycles of an SM each) are enough: with tokens or values as their rows 8 query
// heads fill the columns, and the tensor pipe is 10 % busy at 4.4 TB/s. The tile instructions of an SM want 64 or 128
// rows of one operand and its accumulators outside the registers; they would pay for latent vectors with 64 heads and more,
// where the wide kernel below is bound by its instructions.
//
// Measured on B200, us of the GPU a call with cold L2 (calls back to back in a graph; TB/s of the cache's bytes and the results):
//   1 request of 131072 tokens, 8 key heads of 128, 4 query heads each, bfloat16        86.7   6.19   (90 in a run of seconds)
//   64 requests of up to 4096 tokens, as above                                          31.8   4.36
//   64 requests of 2048 tokens, as above                                                91     5.88
//   1000 requests of up to 100 tokens, as above                                         49.0   2.14
//   1 request of 256 tokens, as above                                                    7.1   0.15   a chain of trips to memory
//   128 requests of up to 8192 tokens, 1 key head of 128, 8 query heads, half           19.8   2.74
//   32 requests of up to 4000 tokens, a latent vector of 320, 16 query heads            18.5   0.46
//   64 requests of up to 8192 tokens, a latent vector of 576, 16 query heads            43.8   1.81
//   17 requests of up to 3001 tokens, 3 key heads of 100, 2 query heads each, float32   16.4   2.01
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kernels.cuh"
#include "kv_paged.h"
#include "kv_values.cuh"

namespace confkv {
namespace kv {

constexpr uint32_t kAttendThreads = 128;
constexpr uint32_t kAttendWarps = kAttendThreads / 32;
constexpr uint32_t kTile = 64;                  // tokens of a tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A row is what one block works on at a time: up to GH query heads, a kernel's own number, of one key head of one request.
struct AttendArgs {
    const char* planes[2];                      // of the layer; one plane: twice the same
    int64_t block_stride, row_stride, page_head_stride;     // bytes, like all strides but lse's and the tables'
    const char* query;
    int64_t query_stride, query_head_stride;
    char* out;
    int64_t out_stride, out_head_stride;
    float* lse;
    int64_t lse_stride;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* lengths;
    float* partial;                             // [2 workers][GH][value_pad]
    float2* partial_sums;                       // [2 workers][GH]: maximum (of base 2), sum
    int4* cut;                                  // [workers]: see cut_of()
    uint32_t requests, blocks, limit, window;
    uint32_t group, chunks;                     // query heads of a key head, rows that they are cut into
    uint32_t rows;                              // of a request
    uint32_t head_dim, value_dim, value_pad;
    float scale;                                // times log2 e: exponents are of base 2
    FastDiv by_block, by_chunks;
    FastDiv by_vector;                          // granules of a vector
    uint32_t granule;                           // bytes of a copy: 16, where SMALL 8 or 4
    Cutting cutting;
    uint32_t cut_by_row;                        // the rows are few
    uint32_t workers;                           // at most
};

// ------------------------------------------------------------------ parts
//
// The rows' units (tiles, and some for a row's beginning and end), one row behind the other, are cut into equal parts, one a worker
// (a block): few long rows and many short ones keep all SMs busy alike, whatever the lengths, which only the device
// knows. A worker that has a whole row writes its result; of a row that is cut each worker writes what it has of it, into its place 1
// where the row begins in its part and into its place 0 where it goes on there, and join_kernel puts them together.

struct PartShared {
    uint32_t warp[8], rest[8];
    uint32_t found, found_sum;
    Span span;
};

__device__ __forceinline__ Span span_at(const AttendArgs& a, uint32_t r)
{
    return span_of(a.lengths[r], a.limit, a.window);
}

__device__ __forceinline__ uint32_t warp_sum(uint32_t v)
{
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        v += __shfl_xor_sync(~0u, v, d);
    }
    return v;
}

// A worker's part, and a row of it with the tiles [first, last) that are the worker's.
struct Part {
    uint64_t begin, end, total, row_begin;      // units; row_begin: the row's first
    uint32_t workers;
    uint32_t request, row, tiles;
    Span span;
    uint32_t first, last;
};

__device__ __forceinline__ void set_row(const AttendArgs& a, Part* p)
{
    p->span = span_at(a, p->request);
    p->tiles = tiles_of(p->span, kTile);
}

// On to the part's next row; false where it has no tiles of any other.
__device__ __forceinline__ bool next_row(const AttendArgs& a, Part* p)
{
    p->row_begin += p->tiles + kRowUnits;
    if (p->row_begin >= p->end) {
        return false;
    }
    if (++p->row == a.rows) {
        p->row = 0;
        // lengths that something else changes meanwhile cost the results, not an address
        if (++p->request >= a.requests) {
            return false;
        }
        set_row(a, p);
    }
    p->first = 0;
    p->last = cut_at(a.cutting, static_cast<int64_t>(p->end - p->row_begin), p->tiles);
    return p->last != 0;
}

// Units of a row of a request.
__device__ __forceinline__ uint32_t units_of(const Span& s) { return tiles_of(s, kTile) + kRowUnits; }

// Every thread gets the same; false for a worker that has no tiles. The units of a row of each request are summed up in 32 bits;
// the first kThreads requests are read once.
template <uint32_t kThreads>
__device__ __forceinline__ bool find_part(const AttendArgs& a, PartShared& s, Part* p)
{
    const uint32_t t = threadIdx.x;
    const Span mine = t < a.requests ? span_at(a, t) : Span{};
    uint32_t n = t < a.requests ? units_of(mine) : 0, up = n, rest = 0;
    for (uint32_t r = t + kThreads; r < a.requests; r += kThreads) {
        rest += units_of(span_at(a, r));
    }
    const auto scan = [&]() {
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t o = __shfl_up_sync(~0u, up, d);
            up += t % 32 >= d ? o : 0;
        }
    };
    scan();
    rest = a.requests > kThreads ? warp_sum(rest) : 0;
    if (t % 32 == 31) {
        s.warp[t / 32] = up;
        s.rest[t / 32] = rest;
    }
    if (t == 0) {
        s.found = s.found_sum = 0;
        s.span = mine;
    }
    __syncthreads();
    uint32_t before = 0, all = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
        before += w < t / 32 ? s.warp[w] : 0;
        all += s.warp[w];
        total += s.rest[w];
    }
    total += all;
    p->total = uint64_t{total} * a.rows;
    p->workers = workers_for(a.cutting, p->total, gridDim.x);
    if (blockIdx.x >= p->workers) {
        return false;
    }
    p->begin = part_start(p->total, p->workers, blockIdx.x);
    p->end = part_start(p->total, p->workers, blockIdx.x + 1);
    // the request that has unit `begin`: the one whose rows begin at or before it
    const auto look = [&](uint32_t r, const Span& span) {
        if (uint64_t{before + up} * a.rows > p->begin && uint64_t{before + up - n} * a.rows <= p->begin) {
            s.found = r;
            s.found_sum = before + up - n;
            s.span = span;
        }
    };
    look(t, mine);
    for (uint32_t from = kThreads; from < a.requests && uint64_t{all} * a.rows <= p->begin; from += kThreads) {
        const uint32_t r = from + t;
        const Span span = r < a.requests ? span_at(a, r) : Span{};
        n = up = r < a.requests ? units_of(span) : 0;
        scan();
        __syncthreads();
        if (t % 32 == 31) {
            s.warp[t / 32] = up;
        }
        __syncthreads();
        before = all;
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 32; ++w) {
            before += w < t / 32 ? s.warp[w] : 0;
            all += s.warp[w];
        }
        look(r, span);
    }
    __syncthreads();
    p->request = s.found;
    p->span = s.span;
    p->tiles = tiles_of(p->span, kTile);
    const uint64_t found_sum = uint64_t{s.found_sum} * a.rows, in = p->begin - found_sum;
    const uint32_t units = p->tiles + kRowUnits;
    p->row = in < (uint64_t{1} << 32) ? static_cast<uint32_t>(in) / units : static_cast<uint32_t>(in / units);
    p->row_begin = found_sum + uint64_t{p->row} * units;
    p->first = cut_at(a.cutting, static_cast<int64_t>(p->begin - p->row_begin), p->tiles);
    p->last = cut_at(a.cutting, static_cast<int64_t>(p->end - p->row_begin), p->tiles);
    return p->last > p->first || next_row(a, p);
}

// The vector of a token: where it starts in its plane, or -1 where its block is not one of the cache's.
__device__ __forceinline__ int64_t token_offset(const AttendArgs& a, const int32_t* table, uint32_t token)
{
    const uint32_t block = quotient(a.by_block, token);
    const int32_t name = table[block];
    return name >= 0 && static_cast<uint32_t>(name) < a.blocks
               ? name * a.block_stride + (token - block * a.by_block.d) * a.row_stride
               : -1;
}

// A row's sums: maximum m (of base 2) of the scores, -infinity where there is none; l, the sum of 2^(s - m). Where all
// scores are -infinity, l is 1 and the row's result NaN, as 0 / 0 is; a row without tokens has l = 0 and the result 0. Other
// pieces with a finite maximum outweigh either.

// The reference that exponents are taken against.
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ float result_factor(float m, float l)
{
    return m == -INFINITY ? (l == 0.0f ? 0.0f : NAN) : 1.0f / l;
}

__device__ __forceinline__ float result_lse(float m, float l)
{
    return m == -INFINITY ? (l == 0.0f ? -INFINITY : NAN) : kLn2 * (m + log2f(l));
}

// What a worker says of its part's last row, for join_kernel: where it begins here and goes on, its request, its row and its last
// worker; else no request.
__device__ __forceinline__ int4 cut_of(const AttendArgs& a, const Part& p)
{
    if (p.first != 0 || p.last == p.tiles) {
        return make_int4(-1, 0, 0, 0);
    }
    return make_int4(static_cast<int>(p.request), static_cast<int>(p.row),
                     static_cast<int>(part_of(p.total, p.workers, p.row_begin + last_units(a.cutting, p.tiles))), 0);
}

// Called by all threads. Where the rows are few join_kernel looks at each of them instead.
__device__ __forceinline__ void note_cut(const AttendArgs& a, const int4& cut)
{
    if (threadIdx.x == 0 && a.cut_by_row == 0) {
        a.cut[blockIdx.x] = cut;
    }
}

// ------------------------------------------------------------------ any type and head size
//
// Each warp takes U tokens at a time. A lane has R values of a vector, in steps of VEC that follow one another (one load, where head size
// and addresses allow), and of GH query heads. The products of GH U scores are summed over the lanes by halving: a lane passes on
// half of its sums at each step and ends with one score (31 exchanges for 32 scores).

// Sums of N values over the warp's lanes: lane i returns the sum of value i % N.
template <int N>
__device__ __forceinline__ float lane_sums(float (&v)[N])
{
    const uint32_t lane = threadIdx.x % 32;
#pragma unroll
    for (int d = 16; d >= N; d /= 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] += __shfl_xor_sync(~0u, v[i], d);
        }
    }
    if constexpr (N > 1) {
#pragma unroll
        for (int d = N / 2; d > 0; d /= 2) {
            const bool high = (lane & d) != 0;
#pragma unroll
            for (int i = 0; i < d; ++i) {
                const float keep = high ? v[i + d] : v[i], send = high ? v[i] : v[i + d];
                v[i] = keep + __shfl_xor_sync(~0u, send, d);
            }
        }
    }
    return v[0];
}

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Values {
    T x[VEC];
};

template <class T, int VEC, int R, int GH, int U, int BLOCKS>
__global__ void __launch_bounds__(kAttendThreads, BLOCKS) attend_any_kernel(const __grid_constant__ AttendArgs a)
{
    constexpr int N = GH * U, STEPS = R / VEC;
    __shared__ PartShared part_shared;
    __shared__ float merge[kAttendWarps][GH][R * 32];
    __shared__ float2 merge_sums[kAttendWarps][GH];
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    Part p;
    if (!find_part<kAttendThreads>(a, part_shared, &p)) {
        note_cut(a, make_int4(-1, 0, 0, 0));
        return;
    }
    const bool one = a.planes[0] == a.planes[1];
    for (;;) {
        const uint32_t tiles = p.last - p.first;
        const uint32_t key_head = quotient(a.by_chunks, p.row), chunk = p.row - key_head * a.by_chunks.d;
        const uint32_t head = key_head * a.group + chunk * GH;              // the row's first query head
        const uint32_t heads = min(static_cast<uint32_t>(GH), a.group - chunk * GH);
        const int32_t* table = a.tables + p.request * a.table_stride;
        const uint32_t from = p.span.first + p.first * kTile;
        const uint32_t to = min(p.span.end, from + tiles * kTile);
        // where the warp's next 32 tokens lie, a token a lane, which is that of the turns to come
        constexpr uint32_t kTurns = 32 / U;
        int64_t offsets = -1;
        uint32_t turn = kTurns;
        const auto find_tokens = [&](uint32_t at) {
            const uint32_t token = at + lane / U * (kAttendWarps * U) + lane % U;
            offsets = token < to ? token_offset(a, table, token) : -1;
            turn = 0;
        };
        find_tokens(from + warp * U);
        float q[GH][R], o[GH][R];
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            const T* query = reinterpret_cast<const T*>(a.query + p.request * a.query_stride + (head + g) * a.query_head_stride);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t d = (lane + i / VEC * 32) * VEC + i % VEC;
                q[g][i] = static_cast<uint32_t>(g) < heads && d < a.head_dim ? to_float(query[d]) * a.scale : 0.0f;
                o[g][i] = 0.0f;
            }
        }
        float m = -INFINITY, l = 0.0f;          // of head lane % N / U; l of token lane % U alone
        bool any = false;
        for (uint32_t at = from + warp * U; at < to; at += kAttendWarps * U) {
            Values<T, VEC> k[U][STEPS], v[U][STEPS];
            uint32_t there = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t offset = __shfl_sync(~0u, offsets, turn * U + u);
                const bool is = offset >= 0;
                there |= is ? 1u << u : 0u;
                const int64_t where = offset + key_head * a.page_head_stride;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const uint32_t d = (lane + i * 32) * VEC;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        k[u][i].x[j] = v[u][i].x[j] = from_float<T>(0.0f);
                    }
                    if (is && d < a.head_dim) {
                        k[u][i] = *reinterpret_cast<const Values<T, VEC>*>(a.planes[0] + where + d * sizeof(T));
                        if (!one) {
                            v[u][i] = *reinterpret_cast<const Values<T, VEC>*>(a.planes[1] + where + d * sizeof(T));
                        }
                    }
                }
            }
            any |= there != 0;
            if (++turn == kTurns) {
                find_tokens(at + kAttendWarps * U);
            }
            float s[N];
#pragma unroll
            for (int g = 0; g < GH; ++g) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float x = 0.0f;
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        x = fmaf(q[g][i], to_float(k[u][i / VEC].x[i % VEC]), x);
                    }
                    s[g * U + u] = x;
                }
            }
            float score = lane_sums<N>(s);
            score = (there >> (lane % U) & 1) != 0 ? score : -INFINITY;
            float top = score;
#pragma unroll
            for (int d = 1; d < U; d *= 2) {
                top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            }
            const float next = fmaxf(m, top), base = reference(next);
            const float weight = exp2f(score - base), fade = exp2f(m - base);
            l = l * fade + weight;
            m = next;
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                const float f = __shfl_sync(~0u, fade, g * U);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    o[g][i] *= f;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float w = __shfl_sync(~0u, weight, g * U + u);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const T y = one ? k[u][i / VEC].x[i % VEC] : v[u][i / VEC].x[i % VEC];
                        o[g][i] = fmaf(w, to_float(y), o[g][i]);
                    }
                }
            }
        }
#pragma unroll
        for (int d = 1; d < U; d *= 2) {
            l += __shfl_xor_sync(~0u, l, d);
        }
        l = m == -INFINITY && l == 0.0f && any ? 1.0f : l;
        if (lane < N && lane % U == 0) {
            merge_sums[warp][lane / U] = make_float2(m, l);
        }
#pragma unroll
        for (int g = 0; g < GH; ++g) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                merge[warp][g][(lane + i / VEC * 32) * VEC + i % VEC] = o[g][i];
            }
        }
        __syncthreads();
        const bool whole = tiles == p.tiles;
        const uint32_t at_place = blockIdx.x * 2 + (p.first == 0 ? 1 : 0);
        for (uint32_t g = warp; g < heads; g += kAttendWarps) {
            float2 part[kAttendWarps];
            float top = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < kAttendWarps; ++w) {
                part[w] = merge_sums[w][g];
                top = fmaxf(top, part[w].x);
            }
            const float base = reference(top);
            float sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kAttendWarps; ++w) {
                // where no piece has a finite maximum, the sums say whether there were tokens
                part[w].x = top == -INFINITY ? 1.0f : exp2f(part[w].x - base);
                sum += part[w].y * part[w].x;
            }
            const float factor = whole ? result_factor(top, sum) : 1.0f;
            T* out = reinterpret_cast<T*>(a.out + p.request * a.out_stride + (head + g) * a.out_head_stride);
            float* partial = a.partial + (uint64_t{at_place} * GH + g) * a.value_pad;
            for (uint32_t d = lane; d < a.value_dim; d += 32) {
                float x = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < kAttendWarps; ++w) {
                    x = fmaf(merge[w][g][d], part[w].x, x);
                }
                if (whole) {
                    out[d] = from_float<T>(x * factor);
                } else {
                    partial[d] = x;
                }
            }
            if (lane == 0) {
                if (!whole) {
                    a.partial_sums[at_place * GH + g] = make_float2(top, sum);
                } else if (a.lse != nullptr) {
                    a.lse[p.request * a.lse_stride + head + g] = result_lse(top, sum);
                }
            }
        }
        const int4 cut = cut_of(a, p);
        if (!next_row(a, &p)) {
            note_cut(a, cut);
            break;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ 16-bit types
//
// A warp takes 16 tokens at a time, in products of 16 x 8 x 16 whose rows are tokens or values and whose columns are query heads: scores =
// K q (K's vectors as they lie), results = V^T p (V's vectors read across), so that 8 query heads fill an instruction's columns and
// nothing is padded to 16 rows. Between the two the weights change places within the warp (movmatrix).
// Each warp has stages of its own, filled by asynchronous copies of 16 bytes two or more tiles ahead, over the ends of rows too:
// no warp waits for another but where a row ends and the four warps' sums are put together.

constexpr uint32_t kWarpTokens = kTile / kAttendWarps;      // 16

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// 16 bytes to shared memory; zeros, and nothing read, where `there` is false.
__device__ __forceinline__ void copy_16(uint32_t to, const char* from, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// 4 or 8 bytes likewise.
__device__ __forceinline__ void copy_small(uint32_t to, const char* from, bool there, uint32_t bytes)
{
    if (bytes == 8) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(there ? 8 : 0) : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
    }
}

__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void copies_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

__device__ __forceinline__ void load_matrices_across(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

__device__ __forceinline__ uint32_t across(uint32_t x)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

template <class T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same_v<T, __half>) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ float power_of_2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Half has no normal numbers below 2^-14: weights of its kernels are held times 2^15, which is as far as the largest, 1, can be raised.
template <class T>
constexpr float kRaised = std::is_same_v<T, __half> ? 15.0f : 0.0f;

// The weight of a score, raised. The maximum goes off first: where floats lie further than 1 apart there (2^24 and more), it raised by
// itself would be rounded to another one, and its own weight to 2^16, more than half holds.
template <class T>
__device__ __forceinline__ float raised_weight(float s, float m)
{
    const float x = s - reference(m);
    if constexpr (std::is_same_v<T, __half>) {
        return power_of_2(x + kRaised<T>);
    } else {
        return power_of_2(x);
    }
}

// Two values in one register, `lo` in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack(float lo, float hi)
{
    uint32_t r;
    if constexpr (std::is_same_v<T, __half>) {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    } else {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    }
    return r;
}

// Two weights as the sums of two of T, so that the products have more of them than T's 8 or 11 bits: each cut to T's bits a little
// below itself, and the rest. Neither is 0 where the weight is not, so that a value's infinity stays one. bfloat16: 2^-15 of the weight is lost. Half: 2^-20,
// or 2^-23 (2^-38 before it was raised) where that is more: both are held at half's least number, 2^-24.
template <class T>
__device__ __forceinline__ void split(float lo, float hi, uint32_t& cut, uint32_t& rest)
{
    if constexpr (std::is_same_v<T, __half>) {
        constexpr float kBelow = 1.0f - 0x1p-12f;
        float c[2], r[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = i == 0 ? lo : hi, least = fminf(x * 0x1p102f, 0x1p-24f);
            const float y = __uint_as_float(__float_as_uint(x * kBelow) & 0xffffe000u);
            c[i] = fmaxf(y, least);
            r[i] = fmaxf(x - y, least);
        }
        cut = pack<T>(c[0], c[1]);
        rest = pack<T>(r[0], r[1]);
    } else {
        constexpr float kBelow = 1.0f - 0x1p-8f;
        const uint32_t x = __float_as_uint(lo * kBelow), y = __float_as_uint(hi * kBelow);
        cut = __byte_perm(x, y, 0x7632);
        rest = pack<T>(lo - __uint_as_float(x & 0xffff0000u), hi - __uint_as_float(y & 0xffff0000u));
    }
}

// DP: values of a vector in shared memory, a multiple of 64, zeros behind head_dim. NT: eights of query heads of a row. ONE: keys
// and values are the same vectors. Vectors are whole chunks of 16 bytes; chunk c of token r lies at place c ^ (r % 8), so
// that eight tokens' chunks of one column lie in different banks.
template <class T, int DP, int NT, bool ONE, int STAGES>
struct MmaShape {
    static constexpr uint32_t kHeads = 8 * NT;
    static constexpr uint32_t kRowBytes = DP * 2;
    static constexpr uint32_t kPlaneBytes = kWarpTokens * kRowBytes;
    static constexpr uint32_t kStageBytes = kPlaneBytes * (ONE ? 1 : 2);
    static constexpr uint32_t kStages = kAttendWarps * STAGES * kStageBytes;
    static constexpr uint32_t kMergeRow = DP + 4;               // floats; heads 2 apart lie 8 banks apart
    static constexpr uint32_t kMergeBytes = 2 * kHeads * kMergeRow * 4;
    static constexpr uint32_t kShared = kStages + kMergeBytes;
    static_assert(kShared + 4096 <= 227 * 1024, "more than a block has");
};

// A warp's way through its block's part, 16 tokens at a step. Of a long row each warp takes a quarter of every tile. With ALONE, where the part
// is long enough for four of them, whole rows of few tiles go to one warp each, in turns, and there is nothing to put together at their
// ends: 1000 requests of up to 100 tokens of 8 key heads take 49 us, and 83 with all rows shared by the warps. The code for it costs
// others 2 to 9 % (64 requests of up to 4096 tokens 32.3 us and 31.1, one of 256 tokens 7.6 and 7.0), so there are two kernels, and calls with rows enough
// for parts of four rows take this one.
template <bool ALONE>
struct Walk {
    Part p;
    uint32_t whole;             // rows met that go to one warp
    uint32_t token, step, left; // the next 16 tokens, those behind them, how many steps are left in the row

    __device__ __forceinline__ bool alone(const AttendArgs& a) const
    {
        return ALONE && p.first == 0 && p.last == p.tiles && p.tiles <= a.cutting.whole_tiles &&
               kAttendWarps * (p.tiles + kRowUnits) <= p.end - p.begin;
    }

    // At the row that p has, if it is one of this warp's, or the next one that is; false where there is none.
    __device__ __forceinline__ bool enter(const AttendArgs& a, uint32_t warp)
    {
        while (alone(a) && whole++ % kAttendWarps != warp) {
            if (!next_row(a, &p)) {
                return false;
            }
        }
        const bool one = alone(a);
        token = p.span.first + (one ? 0 : p.first * kTile + warp * kWarpTokens);
        step = one ? kWarpTokens : kTile;
        left = one ? max(1u, (p.span.end - p.span.first + kWarpTokens - 1) / kWarpTokens) : p.last - p.first;
        return true;
    }

    __device__ __forceinline__ bool next(const AttendArgs& a, uint32_t warp) { return next_row(a, &p) && enter(a, warp); }
};

template <class T, int DP, int NT, bool ONE, int STAGES, int BLOCKS, bool ALONE, bool SMALL>
__global__ void __launch_bounds__(kAttendThreads, BLOCKS) attend_mma_kernel(const __grid_constant__ AttendArgs a)
{
    using Shape = MmaShape<T, DP, NT, ONE, STAGES>;
    constexpr int KT = DP / 16;
    constexpr float kRaise = kRaised<T>;
    constexpr uint32_t GH = Shape::kHeads;
    extern __shared__ __align__(1024) char memory[];
    __shared__ PartShared part_shared;
    constexpr uint32_t kRow = Shape::kMergeRow;
    __shared__ float2 merge_sums[2][kAttendWarps][GH];          // in turns: a warp may write its next row's while others read
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    dev::pdl_release();
    // behind head_dim the stages hold zeros, which no copy touches
    if (a.head_dim != DP) {
        for (uint32_t i = threadIdx.x; i < Shape::kStages / 16; i += kAttendThreads) {
            reinterpret_cast<uint4*>(memory)[i] = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    dev::pdl_wait();
    Part p;
    if (!find_part<kAttendThreads>(a, part_shared, &p)) {
        note_cut(a, make_int4(-1, 0, 0, 0));
        return;
    }
    char* const stages = memory + warp * (STAGES * Shape::kStageBytes);
    const uint32_t stage_base = shared_address(stages);
    float* const merge = reinterpret_cast<float*>(memory + Shape::kStages);    // [2][GH][kRow]
    const uint32_t chunks = a.head_dim / 8;
    const uint32_t tiles16 = (a.head_dim + 15) / 16, value_tiles = (a.value_dim + 15) / 16;

    // what is copied runs ahead of what is computed: the next tile to copy, and the tokens that each tile under way has
    Walk<ALONE> ahead{p, 0, 0, 0, 0};
    bool more_rows = ahead.enter(a, warp);
    Walk<ALONE> now = ahead;
    bool more = more_rows;
    uint32_t tokens_of[STAGES];                 // bit i: token i of this warp's 16 is one
    uint32_t stage_in = 0, stage_out = 0;
    const auto copy_tile = [&]() -> uint32_t {
        uint32_t there = 0;
        if (more_rows) {
            const uint32_t key_head = quotient(a.by_chunks, ahead.p.row);
            const int32_t* table = a.tables + ahead.p.request * a.table_stride;
            const uint32_t token = ahead.token + lane % kWarpTokens;
            int64_t offset = token < ahead.p.span.end ? token_offset(a, table, token) : -1;
            there = __ballot_sync(~0u, offset >= 0) & 0xffffu;
            offset = offset >= 0 ? offset + key_head * a.page_head_stride : 0;
            const uint32_t to = stage_base + stage_in * Shape::kStageBytes;
            const auto copy_chunk = [&](uint32_t r, uint32_t c) {
                const int64_t from = __shfl_sync(~0u, offset, r) + c * 16;
                const uint32_t at = to + r * Shape::kRowBytes + ((c ^ (r % 8)) * 16);
                const bool is = (there >> r & 1) != 0;
                if (r < kWarpTokens) {
                    copy_16(at, a.planes[0] + from, is);
                    if constexpr (!ONE) {
                        copy_16(at + Shape::kPlaneBytes, a.planes[1] + from, is);
                    }
                }
            };
            constexpr uint32_t kChunks = DP / 8;
            if constexpr (SMALL) {
                const uint32_t size = a.granule;
                for (uint32_t k = 0; k < kWarpTokens * a.by_vector.d; k += 32) {
                    const uint32_t r = quotient(a.by_vector, k + lane), at = (k + lane - r * a.by_vector.d) * size;
                    const int64_t from = __shfl_sync(~0u, offset, r) + at;
                    const uint32_t where = to + r * Shape::kRowBytes + (((at / 16) ^ (r % 8)) * 16) + at % 16;
                    const bool is = (there >> r & 1) != 0;
                    if (r < kWarpTokens) {
                        copy_small(where, a.planes[0] + from, is, size);
                        if constexpr (!ONE) {
                            copy_small(where + Shape::kPlaneBytes, a.planes[1] + from, is, size);
                        }
                    }
                }
            } else if (32 % kChunks == 0 && chunks == kChunks) {
#pragma unroll
                for (uint32_t k = 0; k < kWarpTokens * kChunks / 32; ++k) {
                    copy_chunk(k * (32 / kChunks) + lane / kChunks, lane % kChunks);
                }
            } else {
                for (uint32_t k = 0; k < kWarpTokens * chunks; k += 32) {
                    const uint32_t r = quotient(a.by_vector, k + lane);             // 16 and more: behind the last
                    copy_chunk(r, k + lane - r * a.by_vector.d);
                }
            }
            ahead.token += ahead.step;
            if (--ahead.left == 0) {
                more_rows = ahead.next(a, warp);
            }
        }
        copies_end();
        stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
        return there;
    };
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) {
        tokens_of[k] = copy_tile();
    }

    uint32_t turn = 0;
    while (more) {
        p = now.p;
        const bool alone = ALONE && now.step == kWarpTokens;
        const uint32_t key_head = quotient(a.by_chunks, p.row), chunk = p.row - key_head * a.by_chunks.d;
        const uint32_t head = key_head * a.group + chunk * GH;              // the row's first query head
        const uint32_t heads = min(GH, a.group - chunk * GH);
        // q as the second factor: column lane / 4, values 2 (lane % 4) and the next, and 8 further on
        uint32_t q[KT][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t g = n * 8 + lane / 4;
            const char* from = a.query + p.request * a.query_stride + (head + g) * a.query_head_stride + (lane % 4) * 4;
#pragma unroll
            for (int k = 0; k < KT; ++k) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bool is = SMALL ? k * 16 + j * 8 + lane % 4 * 2 < a.head_dim : static_cast<uint32_t>(k * 2 + j) < chunks;
                    q[k][n][j] = g < heads && is
                                     ? *reinterpret_cast<const uint32_t*>(from + k * 32 + j * 16) : 0u;
                }
            }
        }
        float m[NT][2], l[NT][2], o[KT][NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int k = 0; k < KT; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[k][n][i] = 0.0f;
                }
            }
        }
        bool any = false;
        for (; now.left != 0; --now.left) {
            copies_wait<STAGES - 2>();
            __syncwarp();
            tokens_of[STAGES - 1] = copy_tile();
            const uint32_t there = tokens_of[0];
#pragma unroll
            for (int k = 0; k < STAGES - 1; ++k) {
                tokens_of[k] = tokens_of[k + 1];
            }
            const uint32_t keys = stage_base + stage_out * Shape::kStageBytes;
            const uint32_t values = keys + (ONE ? 0 : Shape::kPlaneBytes);
            stage_out = stage_out + 1 == STAGES ? 0 : stage_out + 1;
            if (there == 0) {
                continue;
            }
            any = true;
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            }
            {
                const uint32_t r = lane % 16, c = lane / 16;
                const uint32_t row = keys + r * Shape::kRowBytes;
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    if (static_cast<uint32_t>(k) < tiles16) {
                        uint32_t x[4];
                        load_matrices(x, row + (((2 * k + c) ^ (r % 8)) * 16));
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            multiply<T>(s[n], x, q[k][n][0], q[k][n][1]);
                        }
                    }
                }
            }
            // tokens lane / 4 and lane / 4 + 8, heads 2 (lane % 4) and the next of each eight
            const bool first = (there >> (lane / 4) & 1) != 0, second = (there >> (lane / 4 + 8) & 1) != 0;
            float top[NT][2];
            bool more = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    s[n][j] = first ? s[n][j] * a.scale : -INFINITY;
                    s[n][j + 2] = second ? s[n][j + 2] * a.scale : -INFINITY;
                    float x = fmaxf(s[n][j], s[n][j + 2]);
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) {
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
                    }
                    top[n][j] = fmaxf(m[n][j], x);
                    more |= top[n][j] > m[n][j];
                }
            }
            if (__any_sync(~0u, more)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float fade = power_of_2(m[n][j] - reference(top[n][j]));
                        m[n][j] = top[n][j];
                        l[n][j] *= fade;
#pragma unroll
                        for (int k = 0; k < KT; ++k) {
                            o[k][n][j] *= fade;
                            o[k][n][j + 2] *= fade;
                        }
                    }
                }
            }
            uint32_t w[NT][2], rest[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = raised_weight<T>(s[n][i], m[n][i % 2]);
                    l[n][i % 2] += x[i];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t cut, more_of_it;
                    split<T>(x[2 * h], x[2 * h + 1], cut, more_of_it);
                    w[n][h] = across(cut);
                    rest[n][h] = across(more_of_it);
                }
            }
            {
                const uint32_t r = lane % 8 + lane / 16 * 8, c = lane / 8 % 2;
                const uint32_t row = values + r * Shape::kRowBytes;
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    if (static_cast<uint32_t>(k) < value_tiles) {
                        uint32_t x[4];
                        load_matrices_across(x, row + (((2 * k + c) ^ (r % 8)) * 16));
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            multiply<T>(o[k][n], x, w[n][0], w[n][1]);
                            multiply<T>(o[k][n], x, rest[n][0], rest[n][1]);
                        }
                    }
                }
            }
        }

        const bool whole = p.last - p.first == p.tiles;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) {
                    l[n][j] += __shfl_xor_sync(~0u, l[n][j], d);
                }
                l[n][j] = m[n][j] == -INFINITY && l[n][j] == 0.0f && any ? 1.0f : l[n][j] * power_of_2(-kRaise);
            }
        }
        if (alone) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t g = n * 8 + lane % 4 * 2 + j;
                    if (g < heads) {
                        const float factor = result_factor(m[n][j], l[n][j]) * power_of_2(-kRaise);
                        T* out = reinterpret_cast<T*>(a.out + p.request * a.out_stride + (head + g) * a.out_head_stride);
#pragma unroll
                        for (int k = 0; k < KT; ++k) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t d = k * 16 + h * 8 + lane / 4;
                                if (d < a.value_dim) {
                                    out[d] = from_float<T>(o[k][n][j + 2 * h] * factor);
                                }
                            }
                        }
                        if (lane < 4 && a.lse != nullptr) {
                            a.lse[p.request * a.lse_stride + head + g] = result_lse(m[n][j], l[n][j]);
                        }
                    }
                }
            }
        } else {
            // the four warps' sums together
            float2 (&sums)[kAttendWarps][GH] = merge_sums[turn];
            turn ^= 1;
            if (lane < 4) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        sums[warp][n * 8 + lane * 2 + j] = make_float2(m[n][j], l[n][j]);
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t g = n * 8 + lane % 4 * 2 + j;
                    float top_of_all = -INFINITY;
#pragma unroll
                    for (uint32_t v = 0; v < kAttendWarps; ++v) {
                        top_of_all = fmaxf(top_of_all, sums[v][g].x);
                    }
                    const float f = top_of_all == -INFINITY ? 1.0f : power_of_2(m[n][j] - top_of_all - kRaise);
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        o[k][n][j] *= f;
                        o[k][n][j + 2] *= f;
                    }
                }
            }
            // value lane / 4 (and 8 further on) of each 16, heads as above
            float* const mine = merge + warp % 2 * (GH * kRow) + lane % 4 * 2 * kRow + lane / 4;
            if (warp >= 2) {
#pragma unroll
                for (int k = 0; k < KT; ++k) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mine[(n * 8 + i % 2) * kRow + k * 16 + i / 2 * 8] = o[k][n][i];
                        }
                    }
                }
            }
            __syncthreads();
            if (warp < 2) {
#pragma unroll
                for (int k = 0; k < KT; ++k) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mine[(n * 8 + i % 2) * kRow + k * 16 + i / 2 * 8] += o[k][n][i];
                        }
                    }
                }
            }
            __syncthreads();
            const uint32_t at_place = blockIdx.x * 2 + (p.first == 0 ? 1 : 0);
            for (uint32_t g = warp; g < heads; g += kAttendWarps) {
                float2 part[kAttendWarps];
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < kAttendWarps; ++w) {
                    part[w] = sums[w][g];
                    top = fmaxf(top, part[w].x);
                }
#pragma unroll
                for (uint32_t w = 0; w < kAttendWarps; ++w) {
                    sum += part[w].y * (top == -INFINITY ? 1.0f : power_of_2(part[w].x - top));
                }
                const float factor = whole ? result_factor(top, sum) : 1.0f;
                T* out = reinterpret_cast<T*>(a.out + p.request * a.out_stride + (head + g) * a.out_head_stride);
                float* partial = a.partial + (uint64_t{at_place} * GH + g) * a.value_pad;
                for (uint32_t d = lane; d < a.value_dim; d += 32) {
                    const float x = merge[g * kRow + d] + merge[(GH + g) * kRow + d];
                    if (whole) {
                        out[d] = from_float<T>(x * factor);
                    } else {
                        partial[d] = x;
                    }
                }
                if (lane == 0) {
                    if (!whole) {
                        a.partial_sums[at_place * GH + g] = make_float2(top, sum);
                    } else if (a.lse != nullptr) {
                        a.lse[p.request * a.lse_stride + head + g] = result_lse(top, sum);
                    }
                }
            }
        }
        more = now.next(a, warp);
    }
    copies_wait<0>();
    // a row that is cut was the last one of every warp
    note_cut(a, cut_of(a, p));
}

// ------------------------------------------------------------------ 16-bit types, many query heads
//
// Where more than 8 query heads share a key head, or a vector is long, a block's eight warps share the stages: for the scores a warp takes
// 16 of a tile's 64 tokens and half of the row's 16 NT heads, for the results all tokens and an eighth of the values, so that the
// accumulators stay small (a latent vector's 512 values of 32 heads are 64 registers of a thread, where a warp of its own would need
// 512) and no sums are left to put together at a row's end. Weights and maxima go through shared memory: three
// barriers a tile.

constexpr uint32_t kWideThreads = 256;
constexpr uint32_t kWideWarps = kWideThreads / 32;

template <class T, int DP, int NT, bool ONE, int STAGES>
struct WideShape {
    static constexpr uint32_t kHeads = 16 * NT;
    static constexpr uint32_t kRowBytes = DP * 2;
    static constexpr uint32_t kPlaneBytes = kTile * kRowBytes;
    static constexpr uint32_t kStageBytes = kPlaneBytes * (ONE ? 1 : 2);
    static constexpr uint32_t kQuery = STAGES * kStageBytes;            // where the query heads start
    static constexpr uint32_t kWeightRow = kHeads * 2 + 16;             // bytes; eight tokens' rows lie in different banks
    static constexpr uint32_t kWeightBytes = kTile * kWeightRow;
    static constexpr uint32_t kWeights = kQuery + kHeads * kRowBytes;
    static constexpr uint32_t kShared = kWeights + 2 * kWeightBytes;
    static_assert(kShared + 4096 <= 227 * 1024, "more than a block has");
};

template <class T, int DP, int NT, bool ONE, int STAGES, int BLOCKS>
__global__ void __launch_bounds__(kWideThreads, BLOCKS) attend_wide_kernel(const __grid_constant__ AttendArgs a)
{
    using Shape = WideShape<T, DP, NT, ONE, STAGES>;
    constexpr float kRaise = kRaised<T>;
    constexpr uint32_t GH = Shape::kHeads;
    constexpr int KT = DP / 16;
    constexpr int VS = KT < 8 ? KT : 8, NS = 8 / VS;         // the warps' split of the result: by values, then by heads
    constexpr int VT = (KT + VS - 1) / VS, RT = 2 * NT / NS; // 16-value and 8-head tiles of a warp's share
    static_assert(KT % 2 == 0 && 2 * NT % NS == 0);
    extern __shared__ __align__(1024) char memory[];
    __shared__ PartShared part_shared;
    __shared__ float4 tops[GH];                              // of the four groups of 16 tokens
    __shared__ float4 lane_sums_of[GH];
    __shared__ uint64_t tokens_of[STAGES];                   // bit i of a stage: token i is one
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    dev::pdl_release();
    if (a.head_dim != DP) {
        for (uint32_t i = threadIdx.x; i < Shape::kWeights / 16; i += kWideThreads) {
            reinterpret_cast<uint4*>(memory)[i] = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    dev::pdl_wait();
    Part p;
    if (!find_part<kWideThreads>(a, part_shared, &p)) {
        note_cut(a, make_int4(-1, 0, 0, 0));
        return;
    }
    const uint32_t base = shared_address(memory);
    const uint32_t chunks = a.head_dim / 8;
    const uint32_t tiles16 = (a.head_dim + 15) / 16, value_tiles = (a.value_dim + 15) / 16;

    Part ahead = p;
    bool more_rows = true;
    uint32_t stage_in = 0, stage_out = 0;
    // each warp copies 8 of a tile's 64 vectors
    const auto copy_tile = [&]() {
        if (more_rows) {
            const uint32_t key_head = quotient(a.by_chunks, ahead.row);
            const int32_t* table = a.tables + ahead.request * a.table_stride;
            const uint32_t token = ahead.span.first + ahead.first * kTile + warp * 8 + lane % 8;
            int64_t offset = token < ahead.span.end ? token_offset(a, table, token) : -1;
            const uint32_t there = __ballot_sync(~0u, offset >= 0) & 0xffu;
            offset = offset >= 0 ? offset + key_head * a.page_head_stride : 0;
            if (lane == 0) {
                reinterpret_cast<uint8_t*>(&tokens_of[stage_in])[warp] = static_cast<uint8_t>(there);
            }
            const uint32_t to = base + stage_in * Shape::kStageBytes + warp * 8 * Shape::kRowBytes;
            const auto copy_chunk = [&](uint32_t r, uint32_t c) {
                const int64_t from = __shfl_sync(~0u, offset, r) + c * 16;
                const uint32_t at = to + r * Shape::kRowBytes + ((c ^ r) * 16);
                const bool is = (there >> r & 1) != 0;
                if (r < 8) {
                    copy_16(at, a.planes[0] + from, is);
                    if constexpr (!ONE) {
                        copy_16(at + Shape::kPlaneBytes, a.planes[1] + from, is);
                    }
                }
            };
            constexpr uint32_t kChunks = DP / 8;
            if (32 % kChunks == 0 && chunks == kChunks) {
#pragma unroll
                for (uint32_t k = 0; k < 8 * kChunks / 32; ++k) {
                    copy_chunk(k * (32 / kChunks) + lane / kChunks, lane % kChunks);
                }
            } else {
                for (uint32_t k = 0; k < 8 * chunks; k += 32) {
                    const uint32_t r = quotient(a.by_vector, k + lane);             // 8 and more: behind the last
                    copy_chunk(r, k + lane - r * a.by_vector.d);
                }
            }
            if (++ahead.first == ahead.last) {
                more_rows = next_row(a, &ahead);
            }
        }
        copies_end();
        stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
    };
    // the row's query heads, zeros for those that it does not have: read while the row before is at its last tile, laid down when
    // all warps have that one's scores
    constexpr uint32_t kQueryParts = (GH * DP / 8 + kWideThreads - 1) / kWideThreads;
    uint4 query[kQueryParts];
    const auto read_query = [&](const Part& row) {
        const uint32_t key_head = quotient(a.by_chunks, row.row), chunk = row.row - key_head * a.by_chunks.d;
        const uint32_t heads = min(GH, a.group - chunk * GH);
        const char* from = a.query + row.request * a.query_stride + (key_head * a.group + chunk * GH) * a.query_head_stride;
#pragma unroll
        for (uint32_t k = 0; k < kQueryParts; ++k) {
            const uint32_t i = k * kWideThreads + threadIdx.x, g = quotient(a.by_vector, i), c = i - g * a.by_vector.d;
            query[k] = g < heads ? *reinterpret_cast<const uint4*>(from + g * a.query_head_stride + c * 16) : make_uint4(0, 0, 0, 0);
        }
    };
    const auto write_query = [&]() {
#pragma unroll
        for (uint32_t k = 0; k < kQueryParts; ++k) {
            const uint32_t i = k * kWideThreads + threadIdx.x, g = quotient(a.by_vector, i), c = i - g * a.by_vector.d;
            if (g < GH) {
                *reinterpret_cast<uint4*>(memory + Shape::kQuery + g * Shape::kRowBytes + ((c ^ (g % 8)) * 16)) = query[k];
            }
        }
    };
    read_query(p);
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) {
        copy_tile();
    }
    write_query();

    const uint32_t token_group = warp % 4, head_half = warp / 4;
    const uint32_t value_share = warp % VS, head_share = warp / VS;
    bool more = true;
    while (more) {
        const uint32_t tiles = p.last - p.first;
        const uint32_t key_head = quotient(a.by_chunks, p.row), chunk = p.row - key_head * a.by_chunks.d;
        const uint32_t head = key_head * a.group + chunk * GH;              // the row's first query head
        const uint32_t heads = min(GH, a.group - chunk * GH);
        Part next = p;
        more = next_row(a, &next);
        float m[2 * NT][2], l[NT][2], o[VT][RT][4];         // m of all heads, l of this warp's tokens and half
#pragma unroll
        for (int n = 0; n < 2 * NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            l[n][0] = l[n][1] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < VT; ++v) {
#pragma unroll
            for (int n = 0; n < RT; ++n) {
                o[v][n][0] = o[v][n][1] = o[v][n][2] = o[v][n][3] = 0.0f;
            }
        }
        bool any = false;
        for (uint32_t t = 0; t < tiles; ++t) {
            copies_wait<STAGES - 2>();
            __syncthreads();
            copy_tile();
            const bool query_next = t + 1 == tiles && more;
            if (query_next) {
                read_query(next);
            }
            const uint64_t there = tokens_of[stage_out];
            const uint32_t keys = base + stage_out * Shape::kStageBytes;
            const uint32_t values = keys + (ONE ? 0 : Shape::kPlaneBytes);
            stage_out = stage_out + 1 == STAGES ? 0 : stage_out + 1;
            any |= there != 0;
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            }
            {
                const uint32_t r = token_group * 16 + lane % 16, c = lane / 16;
                const uint32_t row = keys + r * Shape::kRowBytes;
                // two steps of 16 values (NT 1) or two eights of heads (NT 2) in one load
                const uint32_t g = head_half * 8 * NT + (NT == 2 ? lane / 16 * 8 : 0) + lane % 8;
                const uint32_t qc = lane / 8 % 2 + (NT == 1 ? lane / 16 * 2 : 0);
                const uint32_t q_row = base + Shape::kQuery + g * Shape::kRowBytes;
#pragma unroll
                for (int k = 0; k < KT; k += 2) {
                    if (static_cast<uint32_t>(k) < tiles16) {
                        uint32_t x[4], y[4], q[2][4];
                        load_matrices(x, row + (((2 * k + c) ^ (r % 8)) * 16));
                        load_matrices(y, row + (((2 * k + 2 + c) ^ (r % 8)) * 16));
                        load_matrices(q[0], q_row + (((2 * k + qc) ^ (g % 8)) * 16));
                        if constexpr (NT == 1) {
                            multiply<T>(s[0], x, q[0][0], q[0][1]);
                            multiply<T>(s[0], y, q[0][2], q[0][3]);
                        } else {
                            load_matrices(q[1], q_row + (((2 * k + 2 + qc) ^ (g % 8)) * 16));
                            multiply<T>(s[0], x, q[0][0], q[0][1]);
                            multiply<T>(s[1], x, q[0][2], q[0][3]);
                            multiply<T>(s[0], y, q[1][0], q[1][1]);
                            multiply<T>(s[1], y, q[1][2], q[1][3]);
                        }
                    }
                }
            }
            // tokens lane / 4 and lane / 4 + 8 of the warp's 16, heads 2 (lane % 4) and the next of each eight
            const uint32_t mine = static_cast<uint32_t>(there >> (token_group * 16)) & 0xffffu;
            const bool first = (mine >> (lane / 4) & 1) != 0, second = (mine >> (lane / 4 + 8) & 1) != 0;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    s[n][j] = first ? s[n][j] * a.scale : -INFINITY;
                    s[n][j + 2] = second ? s[n][j + 2] * a.scale : -INFINITY;
                    float x = fmaxf(s[n][j], s[n][j + 2]);
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) {
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
                    }
                    if (lane < 4) {
                        reinterpret_cast<float*>(&tops[(head_half * NT + n) * 8 + lane * 2 + j])[token_group] = x;
                    }
                }
            }
            __syncthreads();
            float fade[2 * NT][2];
            bool faded = false;
#pragma unroll
            for (int n = 0; n < 2 * NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float4 x = tops[n * 8 + lane % 4 * 2 + j];
                    const float top = fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), m[n][j]);
                    fade[n][j] = power_of_2(m[n][j] - reference(top));
                    faded |= top > m[n][j];
                    m[n][j] = top;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float ref = head_half != 0 ? m[NT + n][i % 2] : m[n][i % 2];
                    x[i] = raised_weight<T>(s[n][i], ref);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[n][j] = l[n][j] * (head_half != 0 ? fade[NT + n][j] : fade[n][j]) + (x[j] + x[j + 2]);
                }
                const uint32_t at = Shape::kWeights + (token_group * 16 + lane / 4) * Shape::kWeightRow + (head_half * NT + n) * 16 + lane % 4 * 4;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t* const to = reinterpret_cast<uint32_t*>(memory + at + h * 8 * Shape::kWeightRow);
                    split<T>(x[2 * h], x[2 * h + 1], *to, to[Shape::kWeightBytes / 4]);
                }
            }
            if (__any_sync(~0u, faded)) {
#pragma unroll
                for (int n = 0; n < RT; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float f = NS > 1 && head_share != 0 ? fade[(2 * NT - RT) + n][j] : fade[n][j];
#pragma unroll
                        for (int v = 0; v < VT; ++v) {
                            o[v][n][j] *= f;
                            o[v][n][j + 2] *= f;
                        }
                    }
                }
            }
            __syncthreads();
            if (query_next) {
                write_query();
            }
#pragma unroll
            for (int k = 0; k < static_cast<int>(kTile) / 16; ++k) {
                uint32_t w[RT][2], rest[RT][2];
                {
                    const uint32_t r = k * 16 + lane % 16;
                    const uint32_t at = base + Shape::kWeights + r * Shape::kWeightRow + head_share * RT * 16 + lane / 16 * 16;
#pragma unroll
                    for (int n = 0; n < RT; n += 2) {
                        uint32_t x[4];
                        load_matrices_across(x, at + n * 16);
                        w[n][0] = x[0];
                        w[n][1] = x[1];
                        if constexpr (RT > 1) {
                            w[n + 1][0] = x[2];
                            w[n + 1][1] = x[3];
                        }
                        load_matrices_across(x, at + n * 16 + Shape::kWeightBytes);
                        rest[n][0] = x[0];
                        rest[n][1] = x[1];
                        if constexpr (RT > 1) {
                            rest[n + 1][0] = x[2];
                            rest[n + 1][1] = x[3];
                        }
                    }
                }
                const uint32_t r = k * 16 + lane % 8 + lane / 16 * 8, c = lane / 8 % 2;
                const uint32_t row = values + r * Shape::kRowBytes;
#pragma unroll
                for (int v = 0; v < VT; ++v) {
                    const uint32_t tile = value_share + v * VS;
                    if (tile < value_tiles) {
                        uint32_t x[4];
                        load_matrices_across(x, row + (((2 * tile + c) ^ (r % 8)) * 16));
#pragma unroll
                        for (int n = 0; n < RT; ++n) {
                            multiply<T>(o[v][n], x, w[n][0], w[n][1]);
                            multiply<T>(o[v][n], x, rest[n][0], rest[n][1]);
                        }
                    }
                }
            }
        }

        // the sums of the four groups of tokens
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) {
                    l[n][j] += __shfl_xor_sync(~0u, l[n][j], d);
                }
                if (lane < 4) {
                    reinterpret_cast<float*>(&lane_sums_of[(head_half * NT + n) * 8 + lane * 2 + j])[token_group] = l[n][j];
                }
            }
        }
        __syncthreads();
        const bool whole = tiles == p.tiles;
        const uint32_t at_place = blockIdx.x * 2 + (p.first == 0 ? 1 : 0);
#pragma unroll
        for (int n = 0; n < RT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t g = (head_share * RT + n) * 8 + lane % 4 * 2 + j;
                if (g >= heads) {
                    continue;
                }
                const float4 x = lane_sums_of[g];
                const float top = NS > 1 && head_share != 0 ? m[(2 * NT - RT) + n][j] : m[n][j];
                float sum = ((x.x + x.y) + (x.z + x.w)) * power_of_2(-kRaise);
                sum = top == -INFINITY && sum == 0.0f && any ? 1.0f : sum;
                const float factor = (whole ? result_factor(top, sum) : 1.0f) * power_of_2(-kRaise);
                T* out = reinterpret_cast<T*>(a.out + p.request * a.out_stride + (head + g) * a.out_head_stride);
                float* partial = a.partial + (uint64_t{at_place} * GH + g) * a.value_pad;
#pragma unroll
                for (int v = 0; v < VT; ++v) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t d = (value_share + v * VS) * 16 + h * 8 + lane / 4;
                        if (d < a.value_dim) {
                            const float y = o[v][n][j + 2 * h] * factor;
                            if (whole) {
                                out[d] = from_float<T>(y);
                            } else {
                                partial[d] = y;
                            }
                        }
                    }
                }
                if (value_share == 0 && lane < 4) {
                    if (!whole) {
                        a.partial_sums[at_place * GH + g] = make_float2(top, sum);
                    } else if (a.lse != nullptr) {
                        a.lse[p.request * a.lse_stride + head + g] = result_lse(top, sum);
                    }
                }
            }
        }
        if (!more) {
            note_cut(a, cut_of(a, p));
        }
        p = next;
    }
    copies_wait<0>();
}

// ------------------------------------------------------------------ joining
//
// A launch of its own, 3 to 5 us with what it waits for. Joined by the worker that comes last (counted in the workspace, nobody waiting) the pieces cost more,
// since a fence, the count and the pieces are one block's trips to L2 one after the other: 128 requests of up to 8192 tokens 28.6 us,
// and 18.9 at that time with this kernel.
//
// Block (x, g, z): query head g of row x, or of the cut row that begins in worker x's part, if there is one: its first worker's place 1,
// then place 0 of the workers up to its last one. A thread has four values, of share z of them; where a share has fewer
// than the block's threads hold, groups of threads share the pieces. The first pieces are on their way before their weights
// are known: the kernel is a chain of a few trips to L2.

constexpr uint32_t kMostWorkers = 4 * 148;
constexpr uint32_t kJoinAhead = 4;

template <class T>
__global__ void __launch_bounds__(kAttendThreads) join_kernel(const __grid_constant__ AttendArgs a, uint32_t gh)
{
    __shared__ float weights[kMostWorkers];
    __shared__ float tops[kAttendWarps], sums[kAttendWarps];
    __shared__ float4 merge[kAttendThreads];
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t t = threadIdx.x, lane = t % 32, warp = t / 32;
    const uint32_t g = blockIdx.y;
    uint32_t request, row, c, last;
    if (a.cut_by_row != 0) {
        request = blockIdx.x / a.rows;
        row = blockIdx.x - request * a.rows;
        uint32_t all = 0, before = 0;
        for (uint32_t r = t; r < a.requests; r += kAttendThreads) {
            const uint32_t n = units_of(span_at(a, r));
            all += n;
            before += r < request ? n : 0;
        }
        all = warp_sum(all);
        before = warp_sum(before);
        __shared__ uint2 units[kAttendWarps];
        if (lane == 0) {
            units[warp] = make_uint2(all, before);
        }
        __syncthreads();
        uint64_t total = 0, begin = 0;
#pragma unroll
        for (uint32_t w = 0; w < kAttendWarps; ++w) {
            total += units[w].x;
            begin += units[w].y;
        }
        const uint32_t tiles = tiles_of(span_at(a, request), kTile);
        total *= a.rows;
        begin = begin * a.rows + uint64_t{row} * (tiles + kRowUnits);
        const uint32_t workers = workers_for(a.cutting, total, a.workers);
        c = part_of(total, workers, begin + first_units(a.cutting, tiles));
        last = part_of(total, workers, begin + last_units(a.cutting, tiles));
        if (c == last) {
            return;
        }
    } else {
        const int4 cut = a.cut[blockIdx.x];
        if (cut.x < 0) {
            return;
        }
        request = cut.x;
        row = cut.y;
        c = blockIdx.x;
        last = cut.z;
    }
    const uint32_t key_head = quotient(a.by_chunks, row), chunk = row - key_head * a.by_chunks.d;
    if (chunk * gh + g >= a.group) {
        return;
    }
    const uint32_t head = key_head * a.group + chunk * gh + g;
    last = min(last, a.workers - 1);
    if (last < c) {
        return;
    }
    const uint32_t pieces = last - c + 1;
    const auto place = [&](uint32_t k) { return (uint64_t{c + k} * 2 + (k == 0 ? 1 : 0)) * gh + g; };
    // columns of four values, and the groups of threads that share the pieces of one
    const uint32_t all = a.value_pad / 4, share = (all + gridDim.z - 1) / gridDim.z, from = blockIdx.z * share;
    const uint32_t columns = from >= all ? 0 : min(share, all - from);
    if (columns == 0) {
        return;
    }
    const uint32_t groups = columns >= kAttendThreads ? 1 : kAttendThreads / columns;
    const uint32_t column = columns >= kAttendThreads ? t : t % columns, group = columns >= kAttendThreads ? 0 : t / columns;
    const auto value = [&](uint32_t k, uint32_t x) {
        return *reinterpret_cast<const float4*>(a.partial + place(k) * a.value_pad + (from + x) * 4);
    };
    float4 ahead[kJoinAhead];
    const bool works = group < groups && column < columns;
#pragma unroll
    for (uint32_t i = 0; i < kJoinAhead; ++i) {
        const uint32_t k = group + i * groups;
        ahead[i] = works && k < pieces ? value(k, column) : make_float4(0, 0, 0, 0);
    }
    constexpr uint32_t kMine = (kMostWorkers + kAttendThreads - 1) / kAttendThreads;
    float2 x[kMine];
    float top = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const uint32_t k = t + i * kAttendThreads;
        x[i] = k < pieces ? a.partial_sums[place(k)] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, x[i].x);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    }
    if (lane == 0) {
        tops[warp] = top;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kAttendWarps; ++w) {
        top = fmaxf(top, tops[w]);
    }
    const float base = reference(top);
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const uint32_t k = t + i * kAttendThreads;
        if (k < pieces) {
            // where no piece has a finite maximum, the sums say whether there were tokens
            const float w = top == -INFINITY ? 1.0f : exp2f(x[i].x - base);
            weights[k] = w;
            sum += x[i].y * w;
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        sum += __shfl_xor_sync(~0u, sum, d);
    }
    if (lane == 0) {
        sums[warp] = sum;
    }
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kAttendWarps; ++w) {
        sum += sums[w];
    }
    const float factor = result_factor(top, sum);
    T* out = reinterpret_cast<T*>(a.out + request * a.out_stride + head * a.out_head_stride);
    const auto fold = [](float4& s, float w, const float4& v) {
        s.x = fmaf(w, v.x, s.x);
        s.y = fmaf(w, v.y, s.y);
        s.z = fmaf(w, v.z, s.z);
        s.w = fmaf(w, v.w, s.w);
    };
    const auto write = [&](uint32_t x, const float4& s) {
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if ((from + x) * 4 + i < a.value_dim) {
                out[(from + x) * 4 + i] = from_float<T>(v[i] * factor);
            }
        }
    };
    float4 s = make_float4(0, 0, 0, 0);
    if (works) {
#pragma unroll
        for (uint32_t i = 0; i < kJoinAhead; ++i) {
            const uint32_t k = group + i * groups;
            if (k < pieces) {
                fold(s, weights[k], ahead[i]);
            }
        }
#pragma unroll 4
        for (uint32_t k = group + kJoinAhead * groups; k < pieces; k += groups) {
            fold(s, weights[k], value(k, column));
        }
    }
    if (groups > 1) {
        merge[t] = s;
        __syncthreads();
        if (group == 0) {
            for (uint32_t i = 1; i < groups; ++i) {
                fold(s, 1.0f, merge[i * columns + column]);
            }
        }
    }
    if (works && group == 0) {
        write(column, s);
    }
    // vectors of more than 512 values: the columns that are left
    for (uint32_t x = column + kAttendThreads; groups == 1 && x < columns; x += kAttendThreads) {
        float4 more = make_float4(0, 0, 0, 0);
        for (uint32_t k = 0; k < pieces; ++k) {
            fold(more, weights[k], value(k, x));
        }
        write(x, more);
    }
    if (t == 0 && blockIdx.z == 0 && a.lse != nullptr) {
        a.lse[request * a.lse_stride + head] = result_lse(top, sum);
    }
}

}  // namespace kv
}  // namespace confkv
