// Kernels of a paged cache's requests (include/gpu_kv_paged_api.h): block tables and slot maps, and the writing of
// new tokens. Attention is in kv_attend.cuh.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"
#include "kv_paged.h"

namespace confkv {
namespace kv {

// ------------------------------------------------------------------ block tables and slot maps
//
// One launch without workspace: each block scans all requests' changes for itself (8 bytes a request, from L2 but for
// the first block), so that it knows where any name or slot belongs, and then writes its share of them: three sums in front of each request
// (names taken, slots listed, names given back), and a search among them for the request of a name or slot. The sums saturate at
// 2^31 - 1, which is more than any ring or list of slots holds. The bytes are few (2.4 MB for 2000 requests' 290000 slots); a call is a
// launch and a chain of trips to memory: lengths, then a name from a table or the ring, then the slot.
//
// Measured on B200, us of the GPU a call (in a graph): a token for each of 256 requests 3.3; 48 prompts, 18000 slots 4.1; 2000
// requests, 290000 slots 7.1.

constexpr uint32_t kMost = 0x7fffffffu;   // rings and lists of slots are shorter

struct ResizeArgs {
    int32_t* tables;
    int64_t table_stride;
    const int32_t* held;
    const int32_t* lengths;
    int32_t* free;
    const int32_t* cursor;
    int32_t* kept;
    int32_t* cursor_after;
    int64_t* slots;
    int64_t* starts;
    uint32_t capacity, requests, limit, blocks, ring;
    uint32_t per;               // requests of a thread in the scan
    FastDiv by_block;
};

__device__ __forceinline__ uint32_t add_most(uint32_t a, uint32_t b) { return min(a + b, kMost); }

struct Sums {
    uint32_t take, tokens, give;
};

__device__ __forceinline__ Sums add(const Sums& a, const Sums& b)
{
    return Sums{add_most(a.take, b.take), add_most(a.tokens, b.tokens), add_most(a.give, b.give)};
}

__device__ __forceinline__ Sums of_change(const Change& c) { return Sums{c.take, c.tokens, c.give}; }

template <uint32_t THREADS>
struct ResizeShared {
    // exclusive sums in front of each thread's requests, refused ones left out
    uint32_t take[THREADS], tokens[THREADS], give[THREADS];
    Sums warp[THREADS / 32];
    Sums before_refused;        // taken and listed in all
    uint32_t refused;           // the first request that is refused
    uint32_t given;
};

// The last of the threads' sums that is not above i.
template <uint32_t THREADS>
__device__ __forceinline__ uint32_t thread_of(const uint32_t (&sums)[THREADS], uint32_t i)
{
    uint32_t t = 0;
#pragma unroll
    for (uint32_t step = THREADS / 2; step != 0; step /= 2) {
        if (sums[t + step] <= i) {
            t += step;
        }
    }
    return t;
}

__device__ __forceinline__ Change change_at(const ResizeArgs& a, uint32_t r)
{
    return change_of(a.held[r], a.lengths[r], a.limit, a.by_block);
}

__device__ __forceinline__ uint32_t ring_place(uint32_t first, uint32_t n, uint32_t ring)
{
    const uint32_t at = first + n;   // both at most `ring` < 2^31
    return at >= ring ? at - ring : at;
}

template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) resize_kernel(const __grid_constant__ ResizeArgs a)
{
    __shared__ ResizeShared<THREADS> s;
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t / 32;
    const Cursor cursor = cursor_of(a.cursor[0], a.cursor[1], a.ring);
    const uint64_t begin = uint64_t{t} * a.per;
    const uint32_t first = begin < a.requests ? static_cast<uint32_t>(begin) : a.requests;
    const uint32_t last = begin + a.per < a.requests ? static_cast<uint32_t>(begin + a.per) : a.requests;
    Sums mine{};
    for (uint32_t r = first; r < last; ++r) {
        mine = add(mine, of_change(change_at(a, r)));
    }
    Sums up = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const Sums o{__shfl_up_sync(~0u, up.take, d), __shfl_up_sync(~0u, up.tokens, d), __shfl_up_sync(~0u, up.give, d)};
        if (lane >= d) {
            up = add(up, o);
        }
    }
    if (lane == 31) {
        s.warp[warp] = up;
    }
    if (t == 0) {
        s.refused = a.requests;
    }
    __syncthreads();
    Sums sum{};   // in front of this thread's requests
    for (uint32_t w = 0; w < warp; ++w) {
        sum = add(sum, s.warp[w]);
    }
    {
        const Sums o{__shfl_up_sync(~0u, up.take, 1), __shfl_up_sync(~0u, up.tokens, 1), __shfl_up_sync(~0u, up.give, 1)};
        if (lane != 0) {
            sum = add(sum, o);
        }
    }
    // the first request of this thread's that does not fit
    uint32_t refused = a.requests;
    Sums at = sum;
    for (uint32_t r = first; r < last; ++r) {
        const Change c = change_at(a, r);
        const Sums next = add(at, of_change(c));
        if (c.tokens != 0 && (next.take > cursor.count || next.tokens > a.capacity)) {
            refused = r;
            break;
        }
        at = next;
    }
    if (refused < a.requests) {
        atomicMin(&s.refused, refused);
    }
    __syncthreads();
    const uint32_t stop = s.refused;
    if (refused == stop && stop < a.requests) {
        s.before_refused = at;                      // the thread that has it
    } else if (stop == a.requests && t == THREADS - 1) {
        s.before_refused = at;                      // the sums of all
    }
    if (t == THREADS - 1) {
        s.given = add(sum, mine).give;
    }
    __syncthreads();
    const Sums total = s.before_refused;
    s.take[t] = min(sum.take, total.take);
    s.tokens[t] = min(sum.tokens, total.tokens);
    s.give[t] = sum.give;
    __syncthreads();
    const uint32_t given = min(s.given, a.ring - cursor.count);

    // what requests keep, shared out by warps
    if (warp % gridDim.x == blockIdx.x) {
        uint32_t start = s.tokens[t];
        for (uint32_t r = first; r < last; ++r) {
            const Change c = change_at(a, r);
            const bool stays = c.tokens != 0 && r >= stop;
            a.kept[r] = static_cast<int32_t>(stays ? c.held : c.kept);
            if (a.starts != nullptr) {
                a.starts[r] = start;
            }
            start += stays ? 0 : c.tokens;
        }
    }
    if (blockIdx.x == 0 && t == 0) {
        if (a.starts != nullptr) {
            a.starts[a.requests] = total.tokens;
        }
        a.cursor_after[0] = static_cast<int32_t>(a.ring != 0 ? ring_place(cursor.first, total.take, a.ring) : 0);
        a.cursor_after[1] = static_cast<int32_t>(cursor.count - total.take + given);
    }

    // (the bounds in the three searches hold by the sums; they keep every address in its array where something else changes the
    // inputs while the call runs)
    // slots, names taken and names given back in one row, so that their trips to memory do not follow one another in a thread
    const uint32_t listed = a.slots != nullptr ? a.capacity : 0;
    const uint32_t end = a.ring != 0 ? ring_place(cursor.first, cursor.count, a.ring) : 0;
    const uint64_t all = uint64_t{listed} + total.take + given;
    for (uint64_t i = blockIdx.x * THREADS + t; i < all; i += gridDim.x * THREADS) {
        if (i < listed) {
            // the slot of a new token; a block that is taken just now is read from the ring
            const uint32_t n = static_cast<uint32_t>(i);
            int64_t slot = -1;
            if (n < total.tokens) {
                const uint32_t bucket = thread_of(s.tokens, n);
                uint32_t r = bucket * a.per, in = s.tokens[bucket], taken = s.take[bucket];
                Change c = change_at(a, r);
                while (n - in >= c.tokens && r + 1 < a.requests) {
                    in += c.tokens;
                    taken += c.take;
                    c = change_at(a, ++r);
                }
                if (n - in < c.tokens) {
                    const uint32_t token = c.held + (n - in);
                    const uint32_t block = quotient(a.by_block, token), place = taken + (block - c.before);
                    const int32_t name = block < c.before ? a.tables[r * a.table_stride + block]
                                         : place < a.ring ? a.free[ring_place(cursor.first, place, a.ring)] : -1;
                    if (name >= 0 && static_cast<uint32_t>(name) < a.blocks) {
                        slot = int64_t{name} * a.by_block.d + (token - block * a.by_block.d);
                    }
                }
            }
            a.slots[n] = slot;
        } else if (i < uint64_t{listed} + total.take) {
            // the ring's front goes behind the blocks that requests have
            const uint32_t n = static_cast<uint32_t>(i - listed), bucket = thread_of(s.take, n);
            uint32_t r = bucket * a.per, in = s.take[bucket];
            Change c = change_at(a, r);
            while (n - in >= c.take && r + 1 < a.requests) {
                in += c.take;
                c = change_at(a, ++r);
            }
            if (n - in < c.take) {
                a.tables[r * a.table_stride + c.before + (n - in)] = a.free[ring_place(cursor.first, n, a.ring)];
            }
        } else {
            // behind the ring's end
            const uint32_t n = static_cast<uint32_t>(i - listed - total.take), bucket = thread_of(s.give, n);
            uint32_t r = bucket * a.per, in = s.give[bucket];
            Change c = change_at(a, r);
            while (n - in >= c.give && r + 1 < a.requests) {
                in += c.give;
                c = change_at(a, ++r);
            }
            if (n - in < c.give) {
                a.free[ring_place(end, n, a.ring)] = a.tables[r * a.table_stride + (c.before - c.give) + (n - in)];
            }
        }
    }
}

// ------------------------------------------------------------------ new tokens

// A copy: 8191 tokens of 8 heads of 128 bfloat16 take 12.1 us (5.55 TB/s of what is read and written, cold L2), one token 1.1 (a launch).

constexpr uint32_t kAppendThreads = 128;
constexpr uint32_t kAppendUnits = 4;      // granules of a thread

struct AppendArgs {
    const char* source[2];
    int64_t token_stride[2], head_stride[2];        // bytes
    char* plane[2];
    int64_t block_stride, row_stride, page_head_stride;
    const int64_t* slots;
    uint32_t units;                                 // granules of a plane in this launch
    uint32_t cache_slots;
    FastDiv by_vector, by_heads, by_block;          // granules of a vector, heads
};

// Copies granules of the size of G; blockIdx.y is the plane.
template <class G>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a)
{
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t p = blockIdx.y;
    const uint32_t first = blockIdx.x * (kAppendThreads * kAppendUnits) + threadIdx.x;
    G value[kAppendUnits];
    char* to[kAppendUnits];
#pragma unroll
    for (uint32_t k = 0; k < kAppendUnits; ++k) {
        const uint32_t unit = first + k * kAppendThreads;
        to[k] = nullptr;
        if (unit < a.units) {
            const uint32_t vector = quotient(a.by_vector, unit), granule = unit - vector * a.by_vector.d;
            const uint32_t token = quotient(a.by_heads, vector), head = vector - token * a.by_heads.d;
            const int64_t slot = a.slots[token];
            if (slot >= 0 && slot < static_cast<int64_t>(a.cache_slots)) {
                const uint32_t at = static_cast<uint32_t>(slot), block = quotient(a.by_block, at);
                value[k] = *reinterpret_cast<const G*>(a.source[p] + token * a.token_stride[p] + head * a.head_stride[p] +
                                                       granule * sizeof(G));
                to[k] = a.plane[p] + block * a.block_stride + (at - block * a.by_block.d) * a.row_stride +
                        head * a.page_head_stride + granule * sizeof(G);
            }
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < kAppendUnits; ++k) {
        if (to[k] != nullptr) {
            *reinterpret_cast<G*>(to[k]) = value[k];
        }
    }
}

}  // namespace kv
}  // namespace confkv
