// The KV codec's arithmetic up to the rounding to a code; the CPU tests compile it too and check it against
// whole numbers.
#pragma once

#include <cmath>
#include <cstdint>
#include <cstring>

#include "kv_layout.h"

namespace confkv {
namespace kv {

KV_HD uint32_t float_bits(float f)
{
#ifdef __CUDA_ARCH__
    return __float_as_uint(f);
#else
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return u;
#endif
}

KV_HD float bits_float(uint32_t u)
{
#ifdef __CUDA_ARCH__
    return __uint_as_float(u);
#else
    float f;
    std::memcpy(&f, &u, 4);
    return f;
#endif
}

KV_HD float fused(float a, float b, float c) { return fmaf(a, b, c); }
KV_HD double fused(double a, double b, double c) { return fma(a, b, c); }

constexpr uint32_t kInfinity = 0x7f800000u;
constexpr uint32_t kNan = 0x7fffffffu;

// The codes of INT8 and FP8 are roundings of the exact quotient top x / A (top = 127 or 448), and the
// quotient that is computed must not cross a border between two codes. With 2^-E a power of two near
// 1 / A, t = x (top 2^-E) is exact (11 + 7 bits at most for 16-bit caches; where t underflows the code is 0
// anyway), b = A 2^-E is exact, and with y = 1 / b rounded, q0 = t y is within 2^-23 of t / b, of its
// size. The residual t - b q0 is then added back (Markstein's correction step), q = q0 + (t - b q0) y, which leaves one rounding of q and
// some 2^-46. A quotient that is a border itself has few bits, so the residual and then q are
// exact, and the tie goes to even. Any other is at least 2^-19 of its size away from every border: t
// is a whole number T < 2^18 and b a whole number B < 2^11, times powers of two, a border a whole number
// M < 2^8 times one, and T 2^i and M B (or T and M B 2^i) differ by a whole number. float32 caches (T < 2^31,
// B < 2^24, so 2^-32) do the same in double.
//
// Both products of the correction are taken with their signs turned, q = q0 + (b q0 - t)(-y): where x is a zero the residual is +0,
// +0 (-y) = -0, and q0 - 0 is q0 with the sign of x; with t - b q0 it would be q0 + 0, which is +0 for either zero.
template <class F>
struct Divider {
    F c, b, y;
    KV_HD F quotient(float x) const
    {
        const F t = static_cast<F>(x) * c;
        const F q0 = t * y;
        const F r = fused(b, q0, -t);
        return fused(r, -y, q0);
    }
};

// For A = amax, finite. A = 0 gives quotients of 0 for the zeros that it comes from.
template <class F>
KV_HD Divider<F> make_divider(float amax, float top)
{
    Divider<F> d;
    if (amax == 0.0f) {
        d.c = 0;
        d.b = 1;
        d.y = 1;
        return d;
    }
    // E is kept where 2^-E and top 2^-E are normal floats (bfloat16's least A, 2^-133, leaves b = 2^-14)
    int e = static_cast<int>(float_bits(amax) >> 23) - 127;
    e = e < -119 ? -119 : (e > 126 ? 126 : e);
    const float p = bits_float(static_cast<uint32_t>(127 - e) << 23);
    d.c = static_cast<F>(top) * static_cast<F>(p);
    d.b = static_cast<F>(amax) * static_cast<F>(p);
    d.y = static_cast<F>(1) / d.b;
    return d;
}

template <int FMT>
constexpr float kTop = FMT == kInt8 ? 127.0f : 448.0f;

// FLT_MAX / 127 and FLT_MAX / 448, rounded down: no code times a scale overflows.
template <int FMT>
constexpr float kMostScale = FMT == kInt8 ? 0x1.020406p+121f : 0x1.249248p+119f;

// INT8 of 16-bit caches in one product and one rounding a value: with k = 127 / A rounded up, x k + 1.5 2^23 has
// the code of x in its low byte, since it is rounded once, to a whole number, ties to even. k is off by 2^-23 of its
// size at most, and a quotient that is no border is 2^-19 of its size or more away from every one, so that
// only quotients that are borders matter, 254 x = M A for an odd M < 254. 127 then divides M or the whole
// number B that A is times a power of two. M = 127 is the border of 63 and 64, which k from above leads to 64, the
// even one. B = 254, the one multiple of 127 that bfloat16 has, is a power of two times 127: k is
// exact, and the tie goes to even. Half has other multiples of 127; their vectors take the Divider (false), as do vectors
// for which 127 / A is too large for a float.
template <bool HALF>
KV_HD bool int8_factor(float amax, float* k)
{
    const uint32_t bits = float_bits(amax);
    *k = 0.0f;
    if (amax == 0.0f) {
        return true;
    }
    if (amax < 0x1p-119f || (HALF && ((bits >> 13 & 0x3ffu) | 0x400u) % 127u == 0)) {
        return false;
    }
    int e = static_cast<int>(bits >> 23) - 127;
    e = e > 126 ? 126 : e;
    const float p = bits_float(static_cast<uint32_t>(127 - e) << 23);
    const float b = amax * p;                       // 1 to 4
    const float y = 1.0f / b, first = kTop<kInt8> * y;
    // 127 / b, rounded to nearest: the residual is exact; then up where that is below it
    const float near = fused(fused(-b, first, kTop<kInt8>), y, first);
    const float left = fused(-b, near, kTop<kInt8>);
    *k = bits_float(float_bits(near) + (left > 0.0f ? 1u : 0u)) * p;
    return true;
}

// What is added to x k: 1.5 2^23, beside which a float has no bit below 1.
constexpr float kWhole = 12582912.0f;

// A vector's scale; one rounding, to float, which the values read back carry as 2^-24 of their size.
template <int FMT>
KV_HD float scale_of(float amax)
{
    if (amax < 0x1p-100f) {
        return amax / kTop<FMT>;
    }
    // amax / top in three steps, rounded as a division is: the residual of the first is exact
    const float y = 1.0f / kTop<FMT>, q = amax * y;
    return fminf(fused(fused(-q, kTop<FMT>, amax), y, q), kMostScale<FMT>);
}

// A double as the float towards zero, its last bit set where something was lost: a later rounding to
// few bits then goes the way that the double itself would.
KV_HD float round_to_odd(double q)
{
#ifdef __CUDA_ARCH__
    const float f = __double2float_rz(q);
#else
    float f = static_cast<float>(q);
    if (std::fabs(static_cast<double>(f)) > std::fabs(q)) {
        f = bits_float(float_bits(f) - 1u);
    }
#endif
    return static_cast<double>(f) == q ? f : bits_float(float_bits(f) | 1u);
}

KV_HD float for_rounding(float q) { return q; }
KV_HD float for_rounding(double q) { return round_to_odd(q); }

// An MXFP4 block's scale byte e + 127 from the bits of its largest |x|; 255: a value is not finite.
KV_HD uint32_t mx_scale_byte(uint32_t bits)
{
    if (bits >= kInfinity) {
        return 255u;
    }
    const uint32_t biased = bits >> 23;           // floor(log2 A) + 127 of a normal A
    return biased > 2u ? biased - 2u : 0u;
}

// 2^-e of a scale byte below 254; x 2^-e is exact, or so small that its code is 0.
KV_HD float mx_inverse(uint32_t byte) { return bits_float((254u - byte) << 23); }

}  // namespace kv
}  // namespace confkv
