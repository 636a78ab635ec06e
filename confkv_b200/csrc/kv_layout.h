// The KV codec's record layout and index arithmetic, free of CUDA so that the CPU tests compile
// and replay them.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace confkv {
namespace kv {

constexpr int kInt8 = 0, kFp8 = 1, kMxFp4 = 2;          // formats
constexpr int kBf16 = 0, kFp16 = 1, kFp32 = 2;          // cache types
constexpr uint32_t kMagic = 0x3151564bu;                // "KVQ1"
constexpr uint32_t kHeaderBytes = 32;
constexpr uint32_t kMxBlock = 32;                       // values that share an MXFP4 scale
constexpr uint32_t kMaxVectors = 0x7fffffffu;           // of a launch's run: FastDiv's range

KV_HD uint64_t round16(uint64_t n) { return (n + 15) & ~uint64_t{15}; }

KV_HD uint32_t element_bytes(int dtype) { return dtype == kFp32 ? 4u : 2u; }

KV_HD uint32_t code_bytes(int format, uint32_t head_dim)
{
    return format == kMxFp4 ? (head_dim + 1) / 2 : head_dim;
}

KV_HD uint32_t scale_bytes(int format, uint32_t head_dim)
{
    return format == kMxFp4 ? (head_dim + kMxBlock - 1) / kMxBlock : 4u;
}

// Offsets of a record's parts.
struct RecordLayout {
    uint64_t codes_end, scales_at, scales_end, size;
};

KV_HD RecordLayout record_layout(int format, uint32_t head_dim, uint64_t vectors)
{
    RecordLayout r{};
    r.codes_end = kHeaderBytes + vectors * code_bytes(format, head_dim);
    r.scales_at = round16(r.codes_end);
    r.scales_end = r.scales_at + vectors * scale_bytes(format, head_dim);
    r.size = round16(r.scales_end);
    return r;
}

// n / d for n < 2^31 and a fixed d >= 1 by one high product (Granlund and Montgomery's division by an invariant): with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1, n / d = (hi(m n) + n) >> l (the sum stays below 2^32).
struct FastDiv {
    uint32_t d, m, shift;
};

inline FastDiv make_fast_div(uint32_t d)
{
    uint32_t l = 0;
    while ((uint64_t{1} << l) < d) {
        ++l;
    }
    return FastDiv{d, static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << l) - d)) / d + 1), l};
}

KV_HD uint32_t quotient(const FastDiv& f, uint32_t n)
{
#ifdef __CUDA_ARCH__
    return (__umulhi(f.m, n) + n) >> f.shift;
#else
    return (static_cast<uint32_t>((uint64_t{f.m} * n) >> 32) + n) >> f.shift;
#endif
}

// Where a vector of a run belongs: object, then [plane][layer][token][head].
struct VectorIndex {
    uint32_t object, in_object, plane, layer, token, head;
};

KV_HD VectorIndex vector_index(uint32_t v, const FastDiv& by_object, const FastDiv& by_tokens, const FastDiv& by_layers,
                               const FastDiv& by_heads)
{
    VectorIndex x{};
    x.object = quotient(by_object, v);
    x.in_object = v - x.object * by_object.d;
    const uint32_t row = quotient(by_heads, x.in_object);
    x.head = x.in_object - row * by_heads.d;
    const uint32_t pl = quotient(by_tokens, row);
    x.token = row - pl * by_tokens.d;
    x.plane = quotient(by_layers, pl);
    x.layer = pl - x.plane * by_layers.d;
    return x;
}

}  // namespace kv
}  // namespace confkv
