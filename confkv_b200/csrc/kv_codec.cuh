// Kernels of the KV-cache codec (include/gpu_kv_codec_api.h): quantise KV vectors into records and
// read them back.
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

namespace confkv {
namespace kv {

constexpr uint32_t kMaxRuns = 16;      // runs a launch carries in its parameters
constexpr uint32_t kMaxBases = 512;    // planes * layers of a paged cache
constexpr uint32_t kThreads = 256;
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
    FastDiv by_object, by_tokens;       // vectors an object (1 where it has none), tokens
    uint32_t units;                     // of all objects: vectors (one where an object has none) times parts
    uint32_t empty;                     // objects without vectors
    uint32_t passes;                    // units that a group of a tile handles one after another (chunk kernels)
    uint32_t tile_start;                // the run's first tile in the grid
    uint32_t header[4];
};

struct Args {
    FastDiv by_layers, by_heads, by_block;
    FastDiv by_parts;                   // parts that a vector is handled in (chunk kernels)
    uint32_t runs, head_dim, layers, paged;
    uint32_t lg_group;                  // log2 of the lanes a unit has (chunk kernels)
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

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

template <class T>
__device__ __forceinline__ T from_float(float x)
{
    if constexpr (std::is_same_v<T, float>) {
        return x;
    } else if constexpr (std::is_same_v<T, __half>) {
        return __float2half_rn(x);
    } else {
        return __float2bfloat16_rn(x);
    }
}

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

// ------------------------------------------------------- chunks of 16 values
//
// A lane holds chunks of 16 consecutive values: one 32-byte load of a 16-bit cache (two of float32) and one 16- or
// 8-byte store of codes. WIDE: every vector starts at a multiple of 32 bytes and has whole chunks;
// else every vector starts at a multiple of 16 bytes and has whole halves of 8 values.

constexpr uint32_t kChunk = 16;

template <class T>
constexpr uint32_t kChunkWords = kChunk * sizeof(T) / 4;

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

__device__ __forceinline__ void load16(uint32_t* w, const void* p)
{
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
}

__device__ __forceinline__ void store16(void* p, const uint32_t* w)
{
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The words of a chunk; `second`: it has its last 8 values (else zeros stand for them).
template <class T, bool WIDE>
__device__ __forceinline__ void load_chunk(uint32_t* w, const char* p, bool second)
{
    constexpr uint32_t n = kChunkWords<T>;
    if constexpr (WIDE) {
#pragma unroll
        for (uint32_t i = 0; i < n; i += 8) {
            load32(w + i, p + 4 * i);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < n; i += 4) {
            if (i < n / 2 || second) {
                load16(w + i, p + 4 * i);
            }
        }
    }
}

template <class T, bool WIDE>
__device__ __forceinline__ void store_chunk(char* p, const uint32_t* w, bool second)
{
    constexpr uint32_t n = kChunkWords<T>;
    if constexpr (WIDE) {
#pragma unroll
        for (uint32_t i = 0; i < n; i += 8) {
            store32(p + 4 * i, w + i);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < n; i += 4) {
            if (i < n / 2 || second) {
                store16(p + 4 * i, w + i);
            }
        }
    }
}

// Values 2i and 2i + 1 of a chunk.
template <class T>
__device__ __forceinline__ float2 chunk_pair(const uint32_t* w, uint32_t i)
{
    if constexpr (std::is_same_v<T, float>) {
        return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (std::is_same_v<T, __half>) {
        return __half22float2(*reinterpret_cast<const __half2*>(w + i));
    } else {
        return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
}

// The largest |x| of a chunk as the bits of T without the sign (their order is the values', infinity and NaN above).
template <class T>
__device__ __forceinline__ uint32_t chunk_max(const uint32_t* w)
{
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < kChunkWords<T>; ++i) {
        if constexpr (std::is_same_v<T, float>) {
            m = max(m, w[i] & 0x7fffffffu);
        } else {
            asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
        }
    }
    if constexpr (!std::is_same_v<T, float>) {
        m = max(m & 0xffffu, m >> 16);
    }
    return m;
}

// The bits as a float's.
template <class T>
__device__ __forceinline__ uint32_t max_as_float_bits(uint32_t m)
{
    if constexpr (std::is_same_v<T, float>) {
        return m;
    } else if constexpr (std::is_same_v<T, __half>) {
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
    } else {
        return m << 16;
    }
}

// q rounded to a whole number, ties to even, in the low byte of the result: adding 1.5 2^23 (2^52) leaves no
// bit below 1.
__device__ __forceinline__ uint32_t int8_bits(float q) { return __float_as_uint(q + 12582912.0f); }
__device__ __forceinline__ uint32_t int8_bits(double q)
{
    return static_cast<uint32_t>(__double2loint(q + 6755399441055744.0));
}

template <int FMT, class F>
__device__ __forceinline__ uint32_t codes4(const Divider<F>& d, float2 a, float2 b)
{
    const F q0 = d.quotient(a.x), q1 = d.quotient(a.y), q2 = d.quotient(b.x), q3 = d.quotient(b.y);
    if constexpr (FMT == kInt8) {
        const uint32_t lo = __byte_perm(int8_bits(q0), int8_bits(q1), 0x0040);
        const uint32_t hi = __byte_perm(int8_bits(q2), int8_bits(q3), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    } else {
        return e4m3x2(for_rounding(q0), for_rounding(q1)) | e4m3x2(for_rounding(q2), for_rounding(q3)) << 16;
    }
}

// Eight e2m1 codes of x * inverse.
template <class T>
__device__ __forceinline__ uint32_t e2m1_codes8(const uint32_t* w, uint32_t pair, float inverse)
{
    float2 v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        v[i] = chunk_pair<T>(w, pair + i);
        v[i].x *= inverse;
        v[i].y *= inverse;
    }
    uint32_t r;
    asm("{ .reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d}; }"
        : "=r"(r)
        : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
    return r;
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

// A unit is a vector that a group of 2^lg_group lanes holds in R chunks each (INT8, FP8), or a block of 32 values
// that two lanes hold (MXFP4). U units are loaded before the first is worked on.
template <int FMT, class T, bool WIDE, int R, int U>
__global__ void __launch_bounds__(kThreads) quantise_chunk_kernel(const __grid_constant__ Args a)
{
    using F = std::conditional_t<std::is_same_v<T, float>, double, float>;
    constexpr uint32_t words = kChunkWords<T>;
    dev::pdl_release();
    dev::pdl_wait();
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t lg = a.lg_group, lane = threadIdx.x & ((1u << lg) - 1u);
    const uint32_t groups = kThreads >> lg;
    const uint32_t d = a.head_dim;
    uint32_t unit = (blockIdx.x - r.tile_start) * groups * r.passes + (threadIdx.x >> lg);
    for (uint32_t pass = 0; pass < r.passes; pass += U, unit += U * groups) {
        uint32_t w[U][R][words];
        uint32_t in_object[U], part[U], object[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t id = unit + u * groups;
            const uint32_t v = FMT == kMxFp4 ? quotient(a.by_parts, id) : id;
            part[u] = FMT == kMxFp4 ? id - v * a.by_parts.d : 0;
            const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
            in_object[u] = x.in_object;
            object[u] = x.object;
            const char* src = id < r.units && r.empty == 0 ? vector_address(a, r, x) : nullptr;
#pragma unroll
            for (int j = 0; j < R; ++j) {
#pragma unroll
                for (uint32_t i = 0; i < words; ++i) {
                    w[u][j][i] = 0;
                }
                const uint32_t at = (part[u] * 2 + (j << lg) + lane) * kChunk;
                if (src != nullptr && at < d) {
                    load_chunk<T, WIDE>(w[u][j], src + at * sizeof(T), at + kChunk / 2 < d);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                m = max(m, chunk_max<T>(w[u][j]));
            }
            for (uint32_t o = 1; o < 1u << lg; o <<= 1) {
                m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            }
            const uint32_t bits = max_as_float_bits<T>(m);
            if (bits >= kInfinity) {
#pragma unroll
                for (int j = 0; j < R; ++j) {
#pragma unroll
                    for (uint32_t i = 0; i < words; ++i) {
                        w[u][j][i] = 0;
                    }
                }
            }
            if (unit + u * groups >= r.units) {
                continue;                       // no shuffles below
            }
            char* record = r.record + object[u] * r.record_stride;
            if (in_object[u] == 0 && part[u] == 0 && lane == 0) {
                write_frame_of_record(r, record);
            }
            if (r.empty != 0) {
                continue;
            }
            char* codes = record + kHeaderBytes + uint64_t{in_object[u]} * code_bytes(FMT, d);
            if constexpr (FMT == kMxFp4) {
                const uint32_t byte = mx_scale_byte(bits);
                const float inverse = byte == 255u ? 0.0f : mx_inverse(byte);
                const uint32_t at = (part[u] * 2 + lane) * kChunk;
                const uint32_t lo = e2m1_codes8<T>(w[u][0], 0, inverse), hi = e2m1_codes8<T>(w[u][0], 4, inverse);
                if (WIDE) {
                    if (at < d) {
                        *reinterpret_cast<uint2*>(codes + at / 2) = make_uint2(lo, hi);
                    }
                } else {
                    if (at < d) {
                        *reinterpret_cast<uint32_t*>(codes + at / 2) = lo;
                    }
                    if (at + kChunk / 2 < d) {
                        *reinterpret_cast<uint32_t*>(codes + at / 2 + 4) = hi;
                    }
                }
                if (lane == 0) {
                    record[r.scales_at + uint64_t{in_object[u]} * a.by_parts.d + part[u]] = static_cast<char>(byte);
                }
            } else {
                const bool finite = bits < kInfinity;
                const float amax = finite ? __uint_as_float(bits) : 0.0f;
                const Divider<F> div = make_divider<F>(amax, kTop<FMT>);
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    const uint32_t at = ((j << lg) + lane) * kChunk;
                    uint32_t c[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        c[i] = codes4<FMT>(div, chunk_pair<T>(w[u][j], 2 * i), chunk_pair<T>(w[u][j], 2 * i + 1));
                    }
                    if (at < d) {
                        if (WIDE) {
                            store16(codes + at, c);
                        } else {
                            *reinterpret_cast<uint2*>(codes + at) = make_uint2(c[0], c[1]);
                            if (at + kChunk / 2 < d) {
                                *reinterpret_cast<uint2*>(codes + at + 8) = make_uint2(c[2], c[3]);
                            }
                        }
                    }
                }
                if (lane == 0) {
                    reinterpret_cast<float*>(record + r.scales_at)[in_object[u]] =
                        finite ? scale_of<FMT>(amax) : bits_float(kNan);
                }
            }
        }
    }
}

// Four values of the codes in a word (INT8, FP8), before the scale.
template <int FMT>
__device__ __forceinline__ void values4(float* f, uint32_t word)
{
    if constexpr (FMT == kInt8) {
        // 2^23 + 128 + code is a float whose bits are 0x4b0000xx
        const uint32_t u = word ^ 0x80808080u;
        f[0] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - 8388736.0f;
        f[1] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - 8388736.0f;
        f[2] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - 8388736.0f;
        f[3] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - 8388736.0f;
    } else {
        uint32_t lo, hi;
        asm("{ .reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b; }"
            : "=r"(lo), "=r"(hi)
            : "r"(word));
        const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
        f[0] = a.x;
        f[1] = a.y;
        f[2] = b.x;
        f[3] = b.y;
    }
}

// Eight values of the e2m1 codes in a word.
__device__ __forceinline__ void e2m1_values8(float* f, uint32_t word)
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
        const float2 v = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
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

// A unit is a chunk; a thread loads the codes of U before it writes the values of the first.
template <int FMT, class T, bool WIDE, int U>
__global__ void __launch_bounds__(kThreads) dequantise_chunk_kernel(const __grid_constant__ Args a)
{
    constexpr uint32_t words = kChunkWords<T>;
    dev::pdl_release();
    dev::pdl_wait();
    const Run& r = run_of_tile(a, blockIdx.x);
    const uint32_t d = a.head_dim;
    uint32_t unit = (blockIdx.x - r.tile_start) * kThreads * r.passes + threadIdx.x;
    for (uint32_t pass = 0; pass < r.passes; pass += U, unit += U * kThreads) {
        uint32_t c[U][4];
        float scale[U];
        char* dst[U];
        bool second[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t id = unit + u * kThreads;
            dst[u] = nullptr;
            c[u][0] = c[u][1] = c[u][2] = c[u][3] = 0;
            scale[u] = 0.0f;
            second[u] = false;
            if (id >= r.units) {
                continue;
            }
            const uint32_t v = quotient(a.by_parts, id), part = id - v * a.by_parts.d;
            const VectorIndex x = vector_index(v, r.by_object, r.by_tokens, a.by_layers, a.by_heads);
            const char* record = r.record + x.object * r.record_stride;
            const bool good = header_matches(r, record);
            if (x.in_object == 0 && part == 0 && r.ok != nullptr) {
                r.ok[x.object] = good ? 1 : 0;
            }
            if (r.empty != 0) {
                continue;
            }
            char* at = vector_address(a, r, x);
            if (at == nullptr) {
                continue;
            }
            dst[u] = at + part * kChunk * sizeof(T);
            second[u] = part * kChunk + kChunk / 2 < d;
            if (!good) {
                continue;                       // codes and scale 0
            }
            const char* codes = record + kHeaderBytes + uint64_t{x.in_object} * code_bytes(FMT, d);
            if constexpr (FMT == kMxFp4) {
                codes += part * (kChunk / 2);
                if constexpr (WIDE) {
                    const uint2 q = *reinterpret_cast<const uint2*>(codes);
                    c[u][0] = q.x;
                    c[u][1] = q.y;
                } else {
                    c[u][0] = *reinterpret_cast<const uint32_t*>(codes);
                    c[u][1] = second[u] ? *reinterpret_cast<const uint32_t*>(codes + 4) : 0u;
                }
                scale[u] = mx_scale(static_cast<uint8_t>(
                    record[r.scales_at + uint64_t{x.in_object} * scale_bytes(FMT, d) + part / 2]));
            } else {
                codes += part * kChunk;
                if constexpr (WIDE) {
                    load16(c[u], codes);
                } else {
                    const uint2 lo = *reinterpret_cast<const uint2*>(codes);
                    c[u][0] = lo.x;
                    c[u][1] = lo.y;
                    if (second[u]) {
                        const uint2 hi = *reinterpret_cast<const uint2*>(codes + 8);
                        c[u][2] = hi.x;
                        c[u][3] = hi.y;
                    }
                }
                scale[u] = reinterpret_cast<const float*>(record + r.scales_at)[x.in_object];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (dst[u] == nullptr) {
                continue;
            }
            float f[kChunk];
            if constexpr (FMT == kMxFp4) {
                e2m1_values8(f, c[u][0]);
                e2m1_values8(f + 8, c[u][1]);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    values4<FMT>(f + 4 * i, c[u][i]);
                }
            }
            uint32_t w[words];
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i) {
                const float lo = f[2 * i] * scale[u], hi = f[2 * i + 1] * scale[u];
                if constexpr (std::is_same_v<T, float>) {
                    w[2 * i] = __float_as_uint(lo);
                    w[2 * i + 1] = __float_as_uint(hi);
                } else {
                    w[i] = pack2<T>(lo, hi);
                }
            }
            store_chunk<T, WIDE>(dst[u], w, second[u]);
        }
    }
}

}  // namespace kv
}  // namespace confkv
