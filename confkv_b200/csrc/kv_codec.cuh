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
    uint32_t vectors;                   // of all objects; their number where they have none
    uint32_t empty;                     // objects without vectors
    uint32_t tile_start;                // the run's first tile in the grid
    uint32_t header[4];
};

struct Args {
    FastDiv by_layers, by_heads, by_block;
    uint32_t runs, head_dim, layers, paged;
    uint32_t slots;                     // of the paged cache
    int64_t block_stride, row_stride, page_head_stride;   // bytes
    Run run[kMaxRuns];
    char* bases[kMaxBases];             // [plane][layer] of the paged cache
};

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
    if (v >= r.vectors) {
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
    if (v >= r.vectors) {
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

}  // namespace kv
}  // namespace confkv
