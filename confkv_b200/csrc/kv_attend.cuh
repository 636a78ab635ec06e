// Attention of one new token a request over a paged cache (include/gpu_kv_paged_api.h).
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

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

// A row is what one block works on at a time: `heads_of_row` query heads (GH at most) of one key head of one request.
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
    int4* cut;                                  // [workers]: the cut row that begins in a worker's part, its last worker
    uint32_t requests, blocks, limit, window;
    uint32_t group, chunks;                     // query heads of a key head, rows that they are cut into
    uint32_t rows;                              // of a request
    uint32_t head_dim, value_dim, value_pad;
    float scale;                                // times log2 e: exponents are of base 2
    FastDiv by_block, by_chunks;
};

// ------------------------------------------------------------------ parts
//
// The rows' tiles, one row behind the other, are cut into equal parts, one a worker (a block): few long rows and many
// short ones keep all SMs busy alike, whatever the lengths, which only the device knows. A worker that has a whole row writes its
// result; of a row that is cut each worker writes what it has of it, its first row's in place 0 and another's in place 1,
// and join_kernel puts them together.

struct PartShared {
    uint64_t warp[kAttendWarps];
    uint64_t total, found_sum;
    uint32_t found;
};

__device__ __forceinline__ Span span_at(const AttendArgs& a, uint32_t r)
{
    return span_of(a.lengths[r], a.limit, a.window);
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v)
{
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        v += __shfl_xor_sync(~0u, v, d);
    }
    return v;
}

// A worker's part [next, end) and where it begins: tile `tile` of row `row` of request `request`.
struct Part {
    uint64_t next, end, total;
    uint32_t workers;
    uint32_t request, row, tile, tiles;
    Span span;
};

// Every thread gets the same; false for a worker without a part.
template <uint32_t THREADS>
__device__ __forceinline__ bool find_part(const AttendArgs& a, PartShared& s, uint32_t tile, Part* p)
{
    const uint32_t t = threadIdx.x;
    uint64_t sum = 0;
    for (uint32_t r = t; r < a.requests; r += THREADS) {
        sum += tiles_of(span_at(a, r), tile);
    }
    sum = warp_sum(sum);
    if (t % 32 == 0) {
        s.warp[t / 32] = sum;
    }
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 32; ++w) {
        total += s.warp[w];
    }
    p->total = total * a.rows;
    p->workers = p->total < gridDim.x ? static_cast<uint32_t>(p->total) : gridDim.x;
    if (blockIdx.x >= p->workers) {
        return false;
    }
    p->next = part_start(p->total, p->workers, blockIdx.x);
    p->end = part_start(p->total, p->workers, blockIdx.x + 1);
    // the request that has tile `next`: the one whose rows begin at or before it
    uint64_t base = 0;
    for (uint32_t from = 0; from < a.requests; from += THREADS) {
        const uint32_t r = from + t;
        const uint64_t n = r < a.requests ? uint64_t{tiles_of(span_at(a, r), tile)} * a.rows : 0;
        uint64_t up = n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint64_t o = __shfl_up_sync(~0u, up, d);
            up += t % 32 >= d ? o : 0;
        }
        __syncthreads();
        if (t % 32 == 31) {
            s.warp[t / 32] = up;
        }
        __syncthreads();
        uint64_t before = base, all = base;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 32; ++w) {
            before += w < t / 32 ? s.warp[w] : 0;
            all += s.warp[w];
        }
        if (before + up > p->next && before + up - n <= p->next) {
            s.found = r;
            s.found_sum = before + up - n;
        }
        base = all;
        if (all > p->next) {
            break;
        }
    }
    __syncthreads();
    p->request = s.found;
    p->span = span_at(a, p->request);
    p->tiles = tiles_of(p->span, tile);
    const uint64_t in = p->next - s.found_sum;
    p->row = static_cast<uint32_t>(in / p->tiles);
    p->tile = static_cast<uint32_t>(in - uint64_t{p->row} * p->tiles);
    return true;
}

// The next row of a part.
__device__ __forceinline__ void next_row(const AttendArgs& a, uint32_t tile, Part* p)
{
    p->tile = 0;
    if (++p->row == a.rows) {
        p->row = 0;
        ++p->request;
        p->span = span_at(a, p->request);
        p->tiles = tiles_of(p->span, tile);
    }
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

// What a worker says of its part's last row, for join_kernel: where it begins here and goes on, its request, its row, the worker that
// has its last tile, and in which of this worker's places it stands; else no request.
__device__ __forceinline__ void note_cut(const AttendArgs& a, const Part& p, bool cut, uint32_t place)
{
    int4 c = make_int4(-1, 0, 0, 0);
    if (cut) {
        const uint64_t last_tile = p.next - p.tile + p.tiles - 1;
        c = make_int4(static_cast<int>(p.request), static_cast<int>(p.row),
                      static_cast<int>(part_of(p.total, p.workers, last_tile)), static_cast<int>(place));
    }
    a.cut[blockIdx.x] = c;
}

// ------------------------------------------------------------------ any type and head size
//
// Each warp takes U tokens at a time; a lane has values lane, lane + 32, .. of the vectors, R of them, and of GH query heads. The
// products of GH U scores are summed over the lanes by halving: a lane passes on half of its sums at each step and ends with
// one score (31 exchanges for 32 scores).

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

template <class T, int R, int GH, int U>
__global__ void __launch_bounds__(kAttendThreads) attend_any_kernel(const __grid_constant__ AttendArgs a)
{
    constexpr int N = GH * U;
    __shared__ PartShared part_shared;
    __shared__ float merge[kAttendWarps][GH][R * 32];
    __shared__ float2 merge_sums[kAttendWarps][GH];
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    Part p;
    if (!find_part<kAttendThreads>(a, part_shared, kTile, &p)) {
        if (threadIdx.x == 0) {
            note_cut(a, p, false, 0);
        }
        return;
    }
    uint32_t place = 0;
    while (p.next < p.end) {
        const uint64_t left = p.end - p.next;
        const uint32_t tiles = left < p.tiles - p.tile ? static_cast<uint32_t>(left) : p.tiles - p.tile;
        const bool begins = p.tile == 0, ends = p.tile + tiles == p.tiles;
        const uint32_t key_head = quotient(a.by_chunks, p.row), chunk = p.row - key_head * a.by_chunks.d;
        const uint32_t head = key_head * a.group + chunk * GH;              // the row's first query head
        const uint32_t heads = min(static_cast<uint32_t>(GH), a.group - chunk * GH);
        const int32_t* table = a.tables + p.request * a.table_stride;
        float q[GH][R], o[GH][R];
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            const T* from = reinterpret_cast<const T*>(a.query + p.request * a.query_stride + (head + g) * a.query_head_stride);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t d = lane + 32 * i;
                q[g][i] = static_cast<uint32_t>(g) < heads && d < a.head_dim ? to_float(from[d]) * a.scale : 0.0f;
                o[g][i] = 0.0f;
            }
        }
        float m = -INFINITY, l = 0.0f;          // of head lane % N / U; l of token lane % U alone
        bool any = false;
        const uint32_t from = p.span.first + p.tile * kTile;
        const uint32_t to = min(p.span.end, from + tiles * kTile);
        for (uint32_t at = from + warp * U; at < to; at += kAttendWarps * U) {
            int64_t offset[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                offset[u] = at + u < to ? token_offset(a, table, at + u) : -1;
                any |= offset[u] >= 0;
                offset[u] += offset[u] >= 0 ? key_head * a.page_head_stride : 0;
            }
            float k[U][R], v[U][R];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const uint32_t d = lane + 32 * i;
                    const bool there = offset[u] >= 0;
                    k[u][i] = there && d < a.head_dim ? to_float(reinterpret_cast<const T*>(a.planes[0] + offset[u])[d]) : 0.0f;
                    v[u][i] = there && d < a.value_dim ? to_float(reinterpret_cast<const T*>(a.planes[1] + offset[u])[d]) : 0.0f;
                }
            }
            float s[N];
#pragma unroll
            for (int g = 0; g < GH; ++g) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float x = 0.0f;
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        x = fmaf(q[g][i], k[u][i], x);
                    }
                    s[g * U + u] = x;
                }
            }
            float score = lane_sums<N>(s);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                score = lane % U == u && offset[u] < 0 ? -INFINITY : score;
            }
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
                        o[g][i] = fmaf(w, v[u][i], o[g][i]);
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
                merge[warp][g][lane + 32 * i] = o[g][i];
            }
        }
        __syncthreads();
        const bool whole = begins && ends;
        const uint32_t at_place = blockIdx.x * 2 + place;
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
        __syncthreads();
        if (threadIdx.x == 0 && p.next + tiles == p.end) {
            note_cut(a, p, begins && !ends, place);
        }
        p.next += tiles;
        place = 1;
        if (p.next < p.end) {
            next_row(a, kTile, &p);
        }
    }
}

// ------------------------------------------------------------------ joining
//
// Block (c, g): query head g of the row that begins in worker c's part and is cut, if there is one: worker c's last
// place, then the first place of all workers up to the row's last one, in four shares, one a warp.

template <class T>
__global__ void __launch_bounds__(kAttendThreads) join_kernel(const __grid_constant__ AttendArgs a, uint32_t gh)
{
    __shared__ float2 merge_sums[kAttendWarps];
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t c = blockIdx.x, g = blockIdx.y;
    const int4 cut = a.cut[c];
    if (cut.x < 0) {
        return;
    }
    const uint32_t row = cut.y, key_head = quotient(a.by_chunks, row), chunk = row - key_head * a.by_chunks.d;
    if (chunk * gh + g >= a.group) {
        return;
    }
    extern __shared__ float merge[];            // [warps][value_pad]
    const uint32_t head = key_head * a.group + chunk * gh + g;
    const uint32_t pieces = cut.z - c + 1;
    const auto place = [&](uint32_t k) { return (k == 0 ? uint64_t{c} * 2 + cut.w : (uint64_t{c} + k) * 2) * gh + g; };
    float top = -INFINITY;
    for (uint32_t k = threadIdx.x; k < pieces; k += kAttendThreads) {
        top = fmaxf(top, a.partial_sums[place(k)].x);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    }
    if (lane == 0) {
        merge_sums[warp].x = top;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kAttendWarps; ++w) {
        top = fmaxf(top, merge_sums[w].x);
    }
    const float base = reference(top);
    const auto weight = [&](uint32_t k) { return top == -INFINITY ? 1.0f : exp2f(a.partial_sums[place(k)].x - base); };
    float sum = 0.0f;
    for (uint32_t k = warp; k < pieces; k += kAttendWarps) {
        sum += a.partial_sums[place(k)].y * weight(k);
    }
    __syncthreads();
    if (lane == 0) {
        merge_sums[warp].y = sum;
    }
    for (uint32_t d = lane; d < a.value_dim; d += 32) {
        float x = 0.0f;
#pragma unroll 4
        for (uint32_t k = warp; k < pieces; k += kAttendWarps) {
            x = fmaf(a.partial[place(k) * a.value_pad + d], weight(k), x);
        }
        merge[warp * a.value_pad + d] = x;
    }
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kAttendWarps; ++w) {
        sum += merge_sums[w].y;
    }
    const float factor = result_factor(top, sum);
    const uint32_t request = cut.x;
    T* out = reinterpret_cast<T*>(a.out + request * a.out_stride + head * a.out_head_stride);
    for (uint32_t d = threadIdx.x; d < a.value_dim; d += kAttendThreads) {
        float x = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kAttendWarps; ++w) {
            x += merge[w * a.value_pad + d];
        }
        out[d] = from_float<T>(x * factor);
    }
    if (threadIdx.x == 0 && a.lse != nullptr) {
        a.lse[request * a.lse_stride + head] = result_lse(top, sum);
    }
}

}  // namespace kv
}  // namespace confkv
