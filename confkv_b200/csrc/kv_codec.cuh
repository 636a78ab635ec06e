// Kernels of the KV-cache codec (include/gpu_kv_codec_api.h): quantise KV vectors into records and
// read them back.
//
// Both directions are bound by memory: a 16-bit value is 2 bytes on one side and 1 (INT8, FP8) or half a byte (MXFP4)
// on the other, beside one comparison, one product and one rounding. At the 6.55 TB/s of a plain copy
// that is 2.2e12 values a second, for which the SMs have 16 instructions of a lane a value at full clocks
// and 13 at the 1.5 GHz to which the power limit takes them in a run of seconds; so the kernels read each byte once,
// in the widest loads, and spend 7.5 and 6.1 instructions a value (INT8, counted). A call is one launch for up to 16 runs
// of objects of whatever sizes, which travel in the kernel's parameters; there is no workspace and there are no atomics.
//
// Measured on B200, [2, 32, 256, 8, 128] bfloat16 objects (32 MiB), events, L2 cold (quantise / dequantise):
//   32 objects, INT8   231 / 236 us  (7.05 / 6.90 TB/s; 234 to 245 / 238 us in a run of seconds)
//   16 objects, FP8    116 / 120 us  (7.04 / 6.77 TB/s; 127 / 120 us)
//   16 objects, MXFP4   98 / 102 us  (6.96 / 6.68 TB/s; 108 / 101 us)
//   1 object, INT8     9.7 / 9.7 us  (5.25 TB/s: the ramp and the tail of 2048 short blocks)
//   1 token, INT8      2.1 / 2.1 us  (a launch)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "kernels.cuh"
#include "kv_layout.h"
#include "kv_math.h"
#include "kv_values.cuh"

namespace confkv {
namespace kv {

constexpr uint32_t kMaxRuns = 16;      // runs a launch carries in its parameters
constexpr uint32_t kMaxBases = 512;    // planes * layers of a paged cache
constexpr uint32_t kThreads = 128;     // 256: one token 2.7 us for 2.1, the rest within 3 %
constexpr uint32_t kWarps = kThreads / 32;

// Equal objects at equal distances, strides in bytes.
struct Run {
    char* object;
    int64_t object_stride, plane_stride, layer_stride, token_stride, head_stride;
    const int64_t* slots;
    int64_t slots_stride;               // elements
    char* record;
    int64_t record_stride;
    int32_t* ok;
    uint64_t codes_end, scales_at, scales_end, record_bytes;
    FastDiv by_object, by_tokens;       // vectors of an object (1 where it has none), its tokens (or 1)
    uint32_t units;                     // vectors of all objects, one for an object that has none
    uint32_t empty;                     // objects without vectors
    uint32_t tile_start;                // the run's first tile in the grid
    uint32_t header[4];
};

struct Args {
    FastDiv by_layers, by_heads, by_block;
    uint32_t runs, head_dim, layers, paged;
    uint32_t lg_group;                  // log2 of the lanes that share a vector
    uint32_t slots;                     // of the paged cache
    int64_t block_stride, row_stride, page_head_stride;   // bytes
    Run run[kMaxRuns];
    char* bases[kMaxBases];             // [plane][layer] of the paged cache
};

// The run of a tile; runs start at rising tiles.
__device__ __forceinline__ const Run& run_of_tile(const Args& a, uint32_t tile)
{
    uint32_t r = 0;
    while (r + 1 < a.runs && tile >= a.run[r + 1].tile_start) {
        ++r;
    }
    return a.run[r];
}

// The address of a vector, null where its slot is not one of the cache's.
__device__ __forceinline__ char* vector_address(const Args& a, const Run& r, const VectorIndex& x)
{
    if (a.paged == 0) {
        return r.object + x.object * r.object_stride + x.plane * r.plane_stride + x.layer * r.layer_stride +
               x.token * r.token_stride + x.head * r.head_stride;
    }
    const int64_t slot = r.slots[x.object * r.slots_stride + x.token];
    if (slot < 0 || slot >= static_cast<int64_t>(a.slots)) {
        return nullptr;
    }
    const uint32_t s = static_cast<uint32_t>(slot);
    const uint32_t block = quotient(a.by_block, s);
    return a.bases[x.plane * a.layers + x.layer] + block * a.block_stride + (s - block * a.by_block.d) * a.row_stride +
           x.head * a.page_head_stride;
}

// ------------------------------------------------------------------ values

// Two e4m3 codes, `lo` in the low byte; ties to even.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two e2m1 codes in a byte, `lo` in its low half; ties to even, beyond 6 saturated.
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi)
{
    uint32_t r;
    asm("{ .reg .b8 c; cvt.rn.satfinite.e2m1x2.f32 c, %1, %2; cvt.u32.u8 %0, c; }" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The value of an e4m3 code.
__device__ __forceinline__ float e4m3_value(uint32_t code)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(code)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
}

// The value of an e2m1 code: 0, .5, 1, 1.5, 2, 3, 4, 6.
__device__ __forceinline__ float e2m1_value(uint32_t code)
{
    const uint32_t m = code & 7u;
    const float v = m < 4u ? 0.5f * m : (m < 6u ? m - 2.0f : 2.0f * m - 8.0f);
    return (code & 8u) != 0 ? -v : v;
}

// 2^e of a scale byte; NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t byte)
{
    return byte == 255u ? bits_float(kNan) : (byte == 0u ? 0x1p-127f : __uint_as_float(byte << 23));
}

// |x| as an integer: the order of these is that of the values, with infinity and NaN above all.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t warp_max(uint32_t v)
{
    return __reduce_max_sync(0xffffffffu, v);
}

// --------------------------------------------------- one warp a vector
//
// For vectors that no group of lanes holds in its registers: above 2560 values in granules of 16 (float32: 1536), 2048 in ones
// of 8 (reading: 1024), 1024 in ones of 4 and 2 (writing MXFP4 in ones of 4: 2048), 512 in single values. The warp goes
// over an INT8 or FP8 vector twice, the second time out of L1 or L2, and over an MXFP4 one block by block, with loads and stores of single
// values: 1 GiB of bfloat16 vectors of 4096 to INT8 and back 708 / 585 us (2.3 / 2.8 TB/s), to MXFP4 794 / 847 us; 32 chunks to
// INT8, for which there are faster ways, 1157 us.

// The header, and the zero bytes behind the codes and behind the scales.
__device__ __forceinline__ void write_frame_of_record(const Run& r, char* record, uint32_t lane)
{
    if (lane < 8) {
        reinterpret_cast<uint32_t*>(record)[lane] = lane < 4 ? r.header[lane] : 0u;
    }
    if (lane < r.scales_at - r.codes_end) {
        record[r.codes_end + lane] = 0;
    }
    if (lane < r.record_bytes - r.scales_end) {
        record[r.scales_end + lane] = 0;
    }
}

template <int FMT, class T>
__global__ void __launch_bounds__(kThreads) quantise_warp_kernel(const __grid_constant__ Args a)
{
    using F = std::conditional_t<std::is_same_v<T, float>, double, float>;
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t lane = threadIdx.x & 31u;
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t v = (blockIdx.x - r.tile_start) * kWarps + (threadIdx.x >> 5);
    if (v >= r.units) {
        return;
    }
    const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
    char* record = r.record + x.object * r.record_stride;
    if (x.in_object == 0) {
        write_frame_of_record(r, record, lane);
    }
    if (r.empty != 0) {
        return;
    }
    const uint32_t d = a.head_dim;
    const T* src = reinterpret_cast<const T*>(vector_address(a, r, x));
    const uint32_t codes_per_vector = code_bytes(FMT, d);
    uint8_t* codes = reinterpret_cast<uint8_t*>(record) + kHeaderBytes + uint64_t{x.in_object} * codes_per_vector;
    if constexpr (FMT == kMxFp4) {
        const uint32_t blocks = scale_bytes(FMT, d);
        uint8_t* scales = reinterpret_cast<uint8_t*>(record) + r.scales_at + uint64_t{x.in_object} * blocks;
        for (uint32_t k = 0; k < blocks; ++k) {
            const uint32_t i = k * kMxBlock + lane;
            float f = src != nullptr && i < d ? to_float(src[i]) : 0.0f;
            const uint32_t byte = mx_scale_byte(warp_max(magnitude(f)));
            f = byte == 255u ? 0.0f : f * mx_inverse(byte);
            const float next = __shfl_down_sync(0xffffffffu, f, 1);
            if ((lane & 1u) == 0 && i < d) {
                codes[i / 2] = static_cast<uint8_t>(e2m1x2(f, next));
            }
            if (lane == 0) {
                scales[k] = static_cast<uint8_t>(byte);
            }
        }
    } else {
        uint32_t m = 0;
        for (uint32_t i = lane; i < d && src != nullptr; i += 32) {
            m = max(m, magnitude(to_float(src[i])));
        }
        m = warp_max(m);
        const bool finite = m < kInfinity;
        const float amax = finite ? __uint_as_float(m) : 0.0f;
        const Divider<F> div = make_divider<F>(amax, kTop<FMT>);
        for (uint32_t i = lane; i < d; i += 32) {
            const F q = finite && src != nullptr ? div.quotient(to_float(src[i])) : F(0);
            if constexpr (FMT == kInt8) {
                codes[i] = static_cast<uint8_t>(static_cast<int>(rint(q)));
            } else {
                codes[i] = static_cast<uint8_t>(e4m3x2(for_rounding(q), 0.0f));
            }
        }
        if (lane == 0) {
            reinterpret_cast<float*>(record + r.scales_at)[x.in_object] =
                finite ? scale_of<FMT>(amax) : bits_float(kNan);
        }
    }
}

// Whether a record's header is the one that the run's objects have.
__device__ __forceinline__ bool header_matches(const Run& r, const char* record)
{
    const uint4 h = *reinterpret_cast<const uint4*>(record);
    return h.x == r.header[0] && h.y == r.header[1] && h.z == r.header[2] && h.w == r.header[3];
}

template <int FMT, class T>
__global__ void __launch_bounds__(kThreads) dequantise_warp_kernel(const __grid_constant__ Args a)
{
    dev::pdl_release();
    dev::pdl_wait();
    const uint32_t lane = threadIdx.x & 31u;
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t v = (blockIdx.x - r.tile_start) * kWarps + (threadIdx.x >> 5);
    if (v >= r.units) {
        return;
    }
    const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
    const char* record = r.record + x.object * r.record_stride;
    const bool good = header_matches(r, record);
    if (x.in_object == 0 && lane == 0 && r.ok != nullptr) {
        r.ok[x.object] = good ? 1 : 0;
    }
    if (r.empty != 0) {
        return;
    }
    T* dst = reinterpret_cast<T*>(vector_address(a, r, x));
    if (dst == nullptr) {
        return;
    }
    const uint32_t d = a.head_dim;
    const uint8_t* codes =
        reinterpret_cast<const uint8_t*>(record) + kHeaderBytes + uint64_t{x.in_object} * code_bytes(FMT, d);
    for (uint32_t i = lane; i < d; i += 32) {
        float f = 0.0f;
        if (good) {
            if constexpr (FMT == kMxFp4) {
                const uint8_t* scales =
                    reinterpret_cast<const uint8_t*>(record) + r.scales_at + uint64_t{x.in_object} * scale_bytes(FMT, d);
                f = e2m1_value(codes[i / 2] >> (4 * (i & 1u))) * mx_scale(scales[i / kMxBlock]);
            } else {
                const float s = reinterpret_cast<const float*>(record + r.scales_at)[x.in_object];
                f = (FMT == kInt8 ? static_cast<float>(static_cast<int8_t>(codes[i])) : e4m3_value(codes[i])) * s;
            }
        }
        dst[i] = from_float<T>(f);
    }
}

// ------------------------------------------------------- granules of E values
//
// A group of 2^lg_group lanes shares a vector. It is cut into granules of E consecutive values, and lane i of the
// group holds granules i, i + 2^lg_group, ..., R of them: one load each, of 32 bytes where the layout allows it, and one
// store of E codes. E divides head_dim, and every granule starts at a multiple of min(32, E * sizeof(T)) bytes, so
// that a granule is there as a whole or not at all. One lane holds 64 values of the largest granules (R = 4): the
// address of a vector and its scale are the same work for 16 values as for 64 (32 chunks to INT8 with R = 1, 2, 4 and 8: 350,
// 282, 259 and 370 us). SPLIT (MXFP4 alone, E = 2): values are loaded one by one and the last
// granule may lack its second value, for odd head_dim and for vectors at odd addresses.

template <class T, int E>
constexpr int kGranuleWords = E * sizeof(T) / 4;

__device__ __forceinline__ void load32(uint32_t* w, const void* p)
{
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}

__device__ __forceinline__ void store32(void* p, const uint32_t* w)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// BYTES bytes, a power of two, at a multiple of min(32, BYTES); the upper half of the one word of 2 bytes is 0.
template <int BYTES>
__device__ __forceinline__ void load_bytes(uint32_t* w, const void* p)
{
    if constexpr (BYTES >= 32) {
#pragma unroll
        for (int i = 0; i < BYTES / 32; ++i) {
            load32(w + 8 * i, static_cast<const char*>(p) + 32 * i);
        }
    } else if constexpr (BYTES == 16) {
        const uint4 v = *static_cast<const uint4*>(p);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    } else if constexpr (BYTES == 8) {
        const uint2 v = *static_cast<const uint2*>(p);
        w[0] = v.x;
        w[1] = v.y;
    } else if constexpr (BYTES == 4) {
        w[0] = *static_cast<const uint32_t*>(p);
    } else if constexpr (BYTES == 2) {
        w[0] = *static_cast<const uint16_t*>(p);
    } else {
        w[0] = *static_cast<const uint8_t*>(p);
    }
}

template <int BYTES>
__device__ __forceinline__ void store_bytes(void* p, const uint32_t* w)
{
    if constexpr (BYTES >= 32) {
#pragma unroll
        for (int i = 0; i < BYTES / 32; ++i) {
            store32(static_cast<char*>(p) + 32 * i, w + 8 * i);
        }
    } else if constexpr (BYTES == 16) {
        *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (BYTES == 8) {
        *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (BYTES == 4) {
        *static_cast<uint32_t*>(p) = w[0];
    } else if constexpr (BYTES == 2) {
        *static_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    } else {
        *static_cast<uint8_t*>(p) = static_cast<uint8_t>(w[0]);
    }
}

// The words of a granule; `second`: SPLIT, its second value is there.
template <class T, int E, bool SPLIT>
__device__ __forceinline__ void load_granule(uint32_t* w, const T* p, bool second)
{
    if constexpr (!SPLIT) {
        load_bytes<E * sizeof(T)>(w, p);
    } else if constexpr (sizeof(T) == 4) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
        w[1] = second ? *reinterpret_cast<const uint32_t*>(p + 1) : 0u;
    } else {
        w[0] = *reinterpret_cast<const uint16_t*>(p);
        w[0] |= second ? static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 1)) << 16 : 0u;
    }
}

template <class T, int E, bool SPLIT>
__device__ __forceinline__ void store_granule(T* p, const uint32_t* w, bool second)
{
    if constexpr (!SPLIT) {
        store_bytes<E * sizeof(T)>(p, w);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint32_t*>(p) = w[0];
        if (second) {
            *reinterpret_cast<uint32_t*>(p + 1) = w[1];
        }
    } else {
        *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
        if (second) {
            *reinterpret_cast<uint16_t*>(p + 1) = static_cast<uint16_t>(w[0] >> 16);
        }
    }
}

// Two floats in a register pair and the instructions that take both at once, each rounded as its scalar form is:
// half the instructions where the clock, under the power limit, would have them bound the kernel (with
// Int8ByFactor 284 -> 239 us for 32 chunks in a run of seconds).
struct Pair {
    uint64_t v;
};

__device__ __forceinline__ Pair make_pair(float lo, float hi)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
    return p;
}

__device__ __forceinline__ float2 halves(Pair p)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}

__device__ __forceinline__ Pair mul(Pair a, Pair b)
{
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

__device__ __forceinline__ Pair add(Pair a, Pair b)
{
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

__device__ __forceinline__ Pair fused(Pair a, Pair b, Pair c)
{
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}

// Values 2i and 2i + 1 of a granule's words.
template <class T>
__device__ __forceinline__ float2 floats_of(const uint32_t* w, int i)
{
    if constexpr (std::is_same_v<T, float>) {
        return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (std::is_same_v<T, __half>) {
        return __half22float2(*reinterpret_cast<const __half2*>(w + i));
    } else {
        return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
}

template <class T>
__device__ __forceinline__ Pair pair_of(const uint32_t* w, int i)
{
    const float2 f = floats_of<T>(w, i);
    return make_pair(f.x, f.y);
}

// The larger of m and the largest |x| of some words, as the bits of T without the sign, whose order is that of the
// values with infinity and NaN above all. 16-bit types: one maximum for each half of the word; see halves_max.
template <class T, int WORDS>
__device__ __forceinline__ uint32_t max_of(uint32_t m, const uint32_t* w)
{
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if constexpr (sizeof(T) == 4) {
            m = max(m, w[i] & 0x7fffffffu);
        } else {
            asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
        }
    }
    return m;
}

template <class T>
__device__ __forceinline__ uint32_t halves_max(uint32_t m)
{
    return sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
}

// Those bits as a float's.
template <class T>
__device__ __forceinline__ uint32_t as_float_bits(uint32_t m)
{
    if constexpr (std::is_same_v<T, float>) {
        return m;
    } else if constexpr (std::is_same_v<T, __half>) {
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
    } else {
        return m << 16;
    }
}

// The rules by which a granule's codes come from its values; a rule gives the codes of two values in the low two bytes
// (above them something else).

// INT8 of 16-bit caches: one product and one rounding (int8_factor).
struct Int8ByFactor {
    Pair k, whole;
    __device__ __forceinline__ explicit Int8ByFactor(float factor)
        : k(make_pair(factor, factor)), whole(make_pair(kWhole, kWhole))
    {
    }
    __device__ __forceinline__ uint32_t codes(float2 x) const
    {
        const float2 f = halves(fused(make_pair(x.x, x.y), k, whole));
        return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x0040);
    }
};

// The exact quotient, rounded to a whole number by adding 1.5 2^23 (2^52) or to e4m3: Divider's steps with -t, -c and
// -y, which keep the sign of a zero.
template <int FMT>
struct ByQuotient {
    Pair nc, b, ny;
    __device__ __forceinline__ explicit ByQuotient(const Divider<float>& d)
        : nc(make_pair(-d.c, -d.c)), b(make_pair(d.b, d.b)), ny(make_pair(-d.y, -d.y))
    {
    }
    __device__ __forceinline__ uint32_t codes(float2 x) const
    {
        const Pair nt = mul(make_pair(x.x, x.y), nc);
        const Pair q0 = mul(nt, ny);
        const Pair q = fused(fused(b, q0, nt), ny, q0);
        if constexpr (FMT == kInt8) {
            const float2 f = halves(add(q, make_pair(kWhole, kWhole)));
            return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x0040);
        } else {
            const float2 f = halves(q);
            return e4m3x2(f.x, f.y);
        }
    }
};

template <int FMT>
struct ByDoubleQuotient {
    const Divider<double>& d;
    __device__ __forceinline__ uint32_t codes(float2 x) const
    {
        const double q0 = d.quotient(x.x), q1 = d.quotient(x.y);
        if constexpr (FMT == kInt8) {
            constexpr double whole = 6755399441055744.0;
            return __byte_perm(__double2loint(q0 + whole), __double2loint(q1 + whole), 0x0040);
        } else {
            return e4m3x2(round_to_odd(q0), round_to_odd(q1));
        }
    }
};

// The E codes of a granule, INT8 and FP8.
template <class T, int E, class Rule>
__device__ __forceinline__ void codes_of(uint32_t* c, const uint32_t* w, const Rule& rule)
{
    if constexpr (E >= 4) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            c[i] = __byte_perm(rule.codes(floats_of<T>(w, 2 * i)), rule.codes(floats_of<T>(w, 2 * i + 1)), 0x5410);
        }
    } else {
        c[0] = rule.codes(floats_of<T>(w, 0));
    }
}

// The E codes of a granule, MXFP4, of x * inverse.
template <class T, int E>
__device__ __forceinline__ void mx_codes_of(uint32_t* c, const uint32_t* w, Pair inverse)
{
    if constexpr (E >= 8) {
#pragma unroll
        for (int i = 0; i < E / 8; ++i) {
            float2 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = halves(mul(pair_of<T>(w, 4 * i + k), inverse));
            }
            asm("{ .reg .b8 a, b, c, d;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
                "mov.b32 %0, {a, b, c, d}; }"
                : "=r"(c[i])
                : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
        }
    } else {
        uint32_t byte[2];
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            const float2 v = halves(mul(pair_of<T>(w, k), inverse));
            byte[k] = e2m1x2(v.x, v.y);
        }
        c[0] = E == 4 ? __byte_perm(byte[0], byte[E / 4], 0x0040) : byte[0];
    }
}

// The header and the zero bytes behind codes and scales, by one thread.
__device__ __forceinline__ void write_frame_of_record(const Run& r, char* record)
{
    reinterpret_cast<uint4*>(record)[0] = make_uint4(r.header[0], r.header[1], r.header[2], r.header[3]);
    reinterpret_cast<uint4*>(record)[1] = make_uint4(0, 0, 0, 0);
    for (uint64_t i = r.codes_end; i < r.scales_at; ++i) {
        record[i] = 0;
    }
    for (uint64_t i = r.scales_end; i < r.record_bytes; ++i) {
        record[i] = 0;
    }
}

// LG: lg_group where it is known when compiling, else -1. E is 2 or more (quantise_single_kernel below).
//
// MXFP4: a block's granules are in neighbouring lanes, SPAN in each. SPAN = 1: the group has at least 32 / E lanes;
// else it has 32 / (E * SPAN).
template <int FMT, class T, int E, int R, bool SPLIT, int SPAN, int LG>
__global__ void __launch_bounds__(kThreads) quantise_kernel(const __grid_constant__ Args a)
{
    constexpr int words = kGranuleWords<T, E>;
    dev::pdl_release();
    dev::pdl_wait();
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t lg = LG >= 0 ? static_cast<uint32_t>(LG & 31) : a.lg_group, lane = threadIdx.x & ((1u << lg) - 1u);
    const uint32_t groups = kThreads >> lg;
    const uint32_t d = a.head_dim;
    const uint32_t v = (blockIdx.x - r.tile_start) * groups + (threadIdx.x >> lg);
    const bool mine = v < r.units;
    const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
    const T* src = mine && r.empty == 0 ? reinterpret_cast<const T*>(vector_address(a, r, x)) : nullptr;
    uint32_t w[R][words];
#pragma unroll
    for (int j = 0; j < R; ++j) {
#pragma unroll
        for (int i = 0; i < words; ++i) {
            w[j][i] = 0;
        }
        const uint32_t at = ((j << lg) + lane) * E;
        if (src != nullptr && at < d) {
            load_granule<T, E, SPLIT>(w[j], src + at, at + 1 < d);
        }
    }
    char* record = r.record + x.object * r.record_stride;
    uint8_t* codes = reinterpret_cast<uint8_t*>(record) + kHeaderBytes + uint64_t{x.in_object} * code_bytes(FMT, d);
    if (mine && x.in_object == 0 && lane == 0) {
        write_frame_of_record(r, record);
    }
    const bool write = mine && r.empty == 0;
    if constexpr (FMT == kMxFp4) {
        const uint32_t blocks = scale_bytes(FMT, d);
        uint8_t* scales = reinterpret_cast<uint8_t*>(record) + r.scales_at + uint64_t{x.in_object} * blocks;
#pragma unroll
        for (int first = 0; first < R; first += SPAN) {
            if ((static_cast<uint32_t>(first) << lg) * E >= d) {
                break;                          // of all lanes alike
            }
            uint32_t m = 0;
#pragma unroll
            for (int j = first; j < first + SPAN; ++j) {
                m = max_of<T, words>(m, w[j]);
            }
            m = halves_max<T>(m);
#pragma unroll
            for (uint32_t o = 1; o < kMxBlock / (E * SPAN); o <<= 1) {
                m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            }
            const uint32_t byte = mx_scale_byte(as_float_bits<T>(m));
            const uint32_t keep = byte == 255u ? 0u : ~0u;      // codes 0 beside an infinity or a NaN
            const float scale = mx_inverse(byte);
            const Pair inverse = make_pair(scale, scale);
#pragma unroll
            for (int j = first; j < first + SPAN; ++j) {
                const uint32_t at = ((j << lg) + lane) * E;
                if (write && at < d) {
                    uint32_t c[(E + 7) / 8];
                    mx_codes_of<T, E>(c, w[j], inverse);
#pragma unroll
                    for (int i = 0; i < (E + 7) / 8; ++i) {
                        c[i] &= keep;
                    }
                    store_bytes<E / 2>(codes + at / 2, c);
                    if (at % kMxBlock == 0) {
                        scales[at / kMxBlock] = static_cast<uint8_t>(byte);
                    }
                }
            }
        }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            m = max_of<T, words>(m, w[j]);
        }
        m = halves_max<T>(m);
        for (uint32_t o = 1; o < 1u << lg; o <<= 1) {
            m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        }
        if (!write) {
            return;
        }
        const uint32_t bits = as_float_bits<T>(m);
        const bool finite = bits < kInfinity;
        // codes 0 beside an infinity or a NaN, by a mask: values set to 0 beforehand cost 128 registers and 302 us for 238
        const uint32_t keep = finite ? ~0u : 0u;
        const float amax = finite ? __uint_as_float(bits) : 0.0f;
        const auto write_codes = [&](const auto& rule) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const uint32_t at = ((j << lg) + lane) * E;
                if (at < d) {
                    uint32_t c[(E + 3) / 4];
                    codes_of<T, E>(c, w[j], rule);
#pragma unroll
                    for (int i = 0; i < (E + 3) / 4; ++i) {
                        c[i] &= keep;
                    }
                    store_bytes<E>(codes + at, c);
                }
            }
        };
        if constexpr (sizeof(T) == 4) {
            const Divider<double> div = make_divider<double>(amax, kTop<FMT>);
            write_codes(ByDoubleQuotient<FMT>{div});
        } else if constexpr (FMT == kFp8) {
            write_codes(ByQuotient<FMT>(make_divider<float>(amax, kTop<FMT>)));
        } else {
            float factor;
            if (int8_factor<std::is_same_v<T, __half>>(amax, &factor)) {
                write_codes(Int8ByFactor(factor));
            } else {
                write_codes(ByQuotient<FMT>(make_divider<float>(amax, kTop<FMT>)));
            }
        }
        if (lane == 0) {
            reinterpret_cast<float*>(record + r.scales_at)[x.in_object] =
                finite ? scale_of<FMT>(amax) : bits_float(kNan);
        }
    }
}

// The values of the codes in a word (INT8, FP8), before the scale, in twos.
template <int FMT>
__device__ __forceinline__ void values4(Pair* f, uint32_t word)
{
    if constexpr (FMT == kInt8) {
        // 2^23 + 128 + code is a float whose bits are 0x4b0000xx
        const uint32_t u = word ^ 0x80808080u;
        const Pair bias = make_pair(-8388736.0f, -8388736.0f);
        f[0] = add(make_pair(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)),
                             __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441))), bias);
        f[1] = add(make_pair(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)),
                             __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443))), bias);
    } else {
        uint32_t lo, hi;
        asm("{ .reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b; }"
            : "=r"(lo), "=r"(hi)
            : "r"(word));
        f[0] = pair_of<__half>(&lo, 0);
        f[1] = pair_of<__half>(&hi, 0);
    }
}

// The eight values of the e2m1 codes in a word, in twos.
__device__ __forceinline__ void mx_values8(Pair* f, uint32_t word)
{
    uint32_t h[4];
    asm("{ .reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d; }"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = pair_of<__half>(h, i);
    }
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <int FMT, class T, int E, int R, bool SPLIT, int LG>
__global__ void __launch_bounds__(kThreads) dequantise_kernel(const __grid_constant__ Args a)
{
    constexpr int words = kGranuleWords<T, E>;
    constexpr int codes_bytes = FMT == kMxFp4 ? E / 2 : E;
    dev::pdl_release();
    dev::pdl_wait();
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t lg = LG >= 0 ? static_cast<uint32_t>(LG & 31) : a.lg_group, lane = threadIdx.x & ((1u << lg) - 1u);
    const uint32_t groups = kThreads >> lg;
    const uint32_t d = a.head_dim;
    const uint32_t v = (blockIdx.x - r.tile_start) * groups + (threadIdx.x >> lg);
    if (v >= r.units) {
        return;
    }
    const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
    const char* record = r.record + x.object * r.record_stride;
    // the codes are loaded whatever the header says, so that no load waits for another (one object: 10.3 -> 9.7 us)
    const uint8_t* codes =
        reinterpret_cast<const uint8_t*>(record) + kHeaderBytes + uint64_t{x.in_object} * code_bytes(FMT, d);
    uint32_t c[R][(codes_bytes + 3) / 4];
    uint32_t scale[FMT == kMxFp4 ? R : 1];
    if constexpr (FMT != kMxFp4) {
        scale[0] = r.empty == 0 ? reinterpret_cast<const uint32_t*>(record + r.scales_at)[x.in_object] : 0u;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const uint32_t at = ((j << lg) + lane) * E;
        if (FMT == kMxFp4) {
            scale[j] = 0;
        }
        if (at < d && r.empty == 0) {
            load_bytes<codes_bytes>(c[j], codes + (FMT == kMxFp4 ? at / 2 : at));
            if constexpr (FMT == kMxFp4) {
                scale[j] = static_cast<uint8_t>(
                    record[r.scales_at + uint64_t{x.in_object} * scale_bytes(FMT, d) + at / kMxBlock]);
            }
        }
    }
    T* dst = r.empty == 0 ? reinterpret_cast<T*>(vector_address(a, r, x)) : nullptr;
    const bool good = header_matches(r, record);
    if (x.in_object == 0 && lane == 0 && r.ok != nullptr) {
        r.ok[x.object] = good ? 1 : 0;
    }
    if (dst == nullptr) {
        return;
    }
    const uint32_t keep = good ? ~0u : 0u;      // a foreign record's codes and scales are 0
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const uint32_t at = ((j << lg) + lane) * E;
        if (at < d) {
            const uint32_t bits = scale[FMT == kMxFp4 ? j : 0] & keep;
            const float one = FMT == kMxFp4 ? mx_scale(bits) : __uint_as_float(bits);
            const Pair s = make_pair(one, one);
            Pair f[E > 8 ? E / 2 : 4];
            if constexpr (FMT == kMxFp4) {
#pragma unroll
                for (int i = 0; i < (E + 7) / 8; ++i) {
                    mx_values8(f + 4 * i, c[j][i] & keep);
                }
            } else {
#pragma unroll
                for (int i = 0; i < (E + 3) / 4; ++i) {
                    values4<FMT>(f + 2 * i, c[j][i] & keep);
                }
            }
            uint32_t w[words];
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                const float2 v = halves(mul(f[i], s));
                if constexpr (sizeof(T) == 4) {
                    w[2 * i] = __float_as_uint(v.x);
                    w[2 * i + 1] = __float_as_uint(v.y);
                } else {
                    w[i] = pack2<T>(v.x, v.y);
                }
            }
            store_granule<T, E, SPLIT>(dst + at, w, at + 1 < d);
        }
    }
}

// ------------------------------------------------------ single values
//
// INT8 and FP8 of vectors with an odd head size, or at odd addresses: granules of one value, of which a lane holds R, a
// multiple of 4, in a group of 2^LG lanes. Instructions bound this (a load, a store and a test of the end a value), so
// values are worked on in twos and codes in fours, and LG is constant: 8 objects of head size 65 from bfloat16 to INT8
// and back 88 / 88 us (2.4 TB/s), where the granule kernels with E = 1 took 119 / 113.

template <int FMT, class T, int R, int LG>
__global__ void __launch_bounds__(kThreads) quantise_single_kernel(const __grid_constant__ Args a)
{
    constexpr int words = sizeof(T) == 4 ? R : R / 2;
    constexpr uint32_t lanes = 1u << LG;
    dev::pdl_release();
    dev::pdl_wait();
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t lane = threadIdx.x & (lanes - 1u);
    const uint32_t v = (blockIdx.x - r.tile_start) * (kThreads / lanes) + (threadIdx.x >> LG);
    const bool mine = v < r.units;
    const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
    const T* src = mine && r.empty == 0 ? reinterpret_cast<const T*>(vector_address(a, r, x)) : nullptr;
    // this lane's values: those at lane + j * lanes below the head size
    const uint32_t left = lane < a.head_dim ? a.head_dim - lane : 0u;
    const uint32_t there = src != nullptr ? left : 0u;
    src += lane;
    uint32_t w[words];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        uint32_t one = 0;
        if (j * lanes < there) {
            load_bytes<sizeof(T)>(&one, src + j * lanes);
        }
        if constexpr (sizeof(T) == 4) {
            w[j] = one;
        } else {
            w[j / 2] = j % 2 == 0 ? one : __byte_perm(w[j / 2], one, 0x5410);
        }
    }
    uint32_t m = halves_max<T>(max_of<T, words>(0, w));
#pragma unroll
    for (uint32_t o = 1; o < lanes; o <<= 1) {
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    if (!mine) {
        return;
    }
    char* record = r.record + x.object * r.record_stride;
    if (x.in_object == 0 && lane == 0) {
        write_frame_of_record(r, record);
    }
    if (r.empty != 0) {
        return;
    }
    uint8_t* codes = reinterpret_cast<uint8_t*>(record) + kHeaderBytes + uint64_t{x.in_object} * a.head_dim + lane;
    const uint32_t bits = as_float_bits<T>(m);
    const bool finite = bits < kInfinity;
    const uint32_t keep = finite ? ~0u : 0u;
    const float amax = finite ? __uint_as_float(bits) : 0.0f;
    const auto write_codes = [&](const auto& rule) {
#pragma unroll
        for (int j = 0; j < R; j += 2) {
            const uint32_t c = rule.codes(floats_of<T>(w, j / 2)) & keep;
            if (j * lanes < left) {
                codes[j * lanes] = static_cast<uint8_t>(c);
            }
            if ((j + 1) * lanes < left) {
                codes[(j + 1) * lanes] = static_cast<uint8_t>(c >> 8);
            }
        }
    };
    if constexpr (sizeof(T) == 4) {
        const Divider<double> div = make_divider<double>(amax, kTop<FMT>);
        write_codes(ByDoubleQuotient<FMT>{div});
    } else if constexpr (FMT == kFp8) {
        write_codes(ByQuotient<FMT>(make_divider<float>(amax, kTop<FMT>)));
    } else {
        float factor;
        if (int8_factor<std::is_same_v<T, __half>>(amax, &factor)) {
            write_codes(Int8ByFactor(factor));
        } else {
            write_codes(ByQuotient<FMT>(make_divider<float>(amax, kTop<FMT>)));
        }
    }
    if (lane == 0) {
        reinterpret_cast<float*>(record + r.scales_at)[x.in_object] = finite ? scale_of<FMT>(amax) : bits_float(kNan);
    }
}

template <int FMT, class T, int R, int LG>
__global__ void __launch_bounds__(kThreads) dequantise_single_kernel(const __grid_constant__ Args a)
{
    constexpr uint32_t lanes = 1u << LG;
    dev::pdl_release();
    dev::pdl_wait();
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t lane = threadIdx.x & (lanes - 1u);
    const uint32_t v = (blockIdx.x - r.tile_start) * (kThreads / lanes) + (threadIdx.x >> LG);
    if (v >= r.units) {
        return;
    }
    const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
    const char* record = r.record + x.object * r.record_stride;
    const uint32_t left = lane < a.head_dim && r.empty == 0 ? a.head_dim - lane : 0u;
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(record) + kHeaderBytes + uint64_t{x.in_object} * a.head_dim + lane;
    const uint32_t bits = r.empty == 0 ? reinterpret_cast<const uint32_t*>(record + r.scales_at)[x.in_object] : 0u;
    uint32_t c[R / 4];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        uint32_t one = 0;
        if (j * lanes < left) {
            one = codes[j * lanes];
        }
        c[j / 4] = j % 4 == 0 ? one : __byte_perm(c[j / 4], one, j % 4 == 1 ? 0x3240 : (j % 4 == 2 ? 0x3410 : 0x4210));
    }
    T* dst = r.empty == 0 ? reinterpret_cast<T*>(vector_address(a, r, x)) : nullptr;
    const bool good = header_matches(r, record);
    if (x.in_object == 0 && lane == 0 && r.ok != nullptr) {
        r.ok[x.object] = good ? 1 : 0;
    }
    if (dst == nullptr) {
        return;
    }
    dst += lane;
    const uint32_t keep = good ? ~0u : 0u;
    const Pair s = make_pair(__uint_as_float(bits & keep), __uint_as_float(bits & keep));
#pragma unroll
    for (int j = 0; j < R; j += 4) {
        Pair f[2];
        values4<FMT>(f, c[j / 4] & keep);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 p = halves(mul(f[i], s));
            if ((j + 2 * i) * lanes < left) {
                dst[(j + 2 * i) * lanes] = from_float<T>(p.x);
            }
            if ((j + 2 * i + 1) * lanes < left) {
                dst[(j + 2 * i + 1) * lanes] = from_float<T>(p.y);
            }
        }
    }
}

}  // namespace kv
}  // namespace confkv
