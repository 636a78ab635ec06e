// Host build of the KV codec's arithmetic (csrc/kv_math.h, kv_layout.h) for tests/test_kv_layout.py.
#include <cstdint>
#include <cstdlib>
#include <initializer_list>

#include "kv_math.h"

namespace kv = confkv::kv;

// One side of a border between two codes, or on it: the sign of top x / A - border, from whole numbers. x = X 2^i,
// A = B 2^j, border = M 2^k, all positive.
static int side(int64_t x, int i, int64_t b, int j, int64_t top, int64_t m, int k)
{
    __int128 left = static_cast<__int128>(top) * x, right = static_cast<__int128>(m) * b;
    const int shift = i - j - k;
    if (shift >= 0) {
        left <<= shift;
    } else {
        right <<= -shift;
    }
    return left > right ? 1 : (left < right ? -1 : 0);
}

// Every quotient of a `bits`-bit whole number by another times 2^-gap, gap up to max_gap: the borders next to the
// quotient that the kernels compute have to be on the same sides of it as of the exact quotient. `step` > 1 visits
// each step-th x. The number of failures.
template <class F>
static uint64_t check_quotients(int format, int bits, int max_gap, int step, int exponent)
{
    const int64_t lo = int64_t{1} << (bits - 1), hi = int64_t{1} << bits;
    const int64_t top = format == kv::kInt8 ? 127 : 448;
    uint64_t bad = 0;
    for (int64_t b = lo; b < hi; b += (step > 1 ? 1 + (b * 7919) % step : 1)) {
        const float amax = std::ldexp(static_cast<float>(b), exponent);
        const kv::Divider<F> div = kv::make_divider<F>(amax, static_cast<float>(top));
        for (int gap = 0; gap <= max_gap; ++gap) {
            for (int64_t x = lo; x < hi; x += (step > 1 ? 1 + (x * 104729 + b) % step : 1)) {
                const float xv = std::ldexp(static_cast<float>(x), exponent - gap);
                if (xv > amax) {
                    break;
                }
                const F q = div.quotient(xv);
                // the border below or at q, and the next: odd multiples of half a step
                int k = -1;
                if (format == kv::kFp8) {
                    int e = std::ilogb(q > 0 ? static_cast<double>(q) : 1e-30);
                    e = e < -6 ? -6 : e;
                    k = e - 3 - 1;
                }
                const double units = std::ldexp(static_cast<double>(q), -k);   // of half steps
                int64_t m = static_cast<int64_t>(std::floor(units));
                m -= (m & 1) == 0 ? 1 : 0;
                for (int64_t border = m; border <= m + 2; border += 2) {
                    if (border < 0) {
                        continue;
                    }
                    const int want = side(x, exponent - gap, b, exponent, top, border, k);
                    const int got = units > border ? 1 : (units < border ? -1 : 0);
                    bad += want != got;
                }
                if (sizeof(F) == 8) {
                    // the float that the conversion to e4m3 gets keeps to the same side of the borders
                    const double odd = std::ldexp(static_cast<double>(kv::for_rounding(q)), -k);
                    for (int64_t border = m; border <= m + 2; border += 2) {
                        bad += border >= 0 && (odd > border) != (units > border);
                        bad += border >= 0 && (odd < border) != (units < border);
                    }
                }
            }
        }
    }
    return bad;
}

// The INT8 codes of check_quotients' quotients by int8_factor, both signs, against whole numbers.
template <bool HALF>
static uint64_t check_int8(int bits, int max_gap, int exponent, uint64_t* slow)
{
    const int64_t lo = int64_t{1} << (bits - 1), hi = int64_t{1} << bits;
    uint64_t bad = 0;
    for (int64_t b = lo; b < hi; ++b) {
        const float amax = std::ldexp(static_cast<float>(b), exponent);
        float k;
        if (!kv::int8_factor<HALF>(amax, &k)) {
            ++*slow;
            continue;
        }
        for (int gap = 0; gap <= max_gap; ++gap) {
            for (int64_t x = lo; x < hi; ++x) {
                const float xv = std::ldexp(static_cast<float>(x), exponent - gap);
                if (xv > amax) {
                    break;
                }
                // 127 x 2^-gap / b rounded to a whole number, ties to even
                const int64_t num = 127 * x, den = b << gap;
                int64_t code = num / den;
                const int64_t twice = 2 * (num - code * den);
                code += twice > den || (twice == den && (code & 1) != 0) ? 1 : 0;
                for (int sign = -1; sign <= 1; sign += 2) {
                    const uint32_t f = kv::float_bits(kv::fused(sign * xv, k, kv::kWhole));
                    bad += static_cast<int8_t>(f & 0xffu) != sign * code;
                }
            }
        }
    }
    return bad;
}

// Zeros of both signs, and values so small that their quotients are zero: the quotients that do not have their sign.
template <class F>
static uint64_t check_signs(int format, int exponent)
{
    uint64_t bad = 0;
    const float top = format == kv::kInt8 ? 127.0f : 448.0f, tiny = kv::bits_float(1);
    for (uint32_t b = 0; b < 256; ++b) {
        const float amax = b == 0 ? 0.0f : std::ldexp(static_cast<float>(b), exponent);
        const kv::Divider<F> div = kv::make_divider<F>(amax, top);
        for (float x : {0.0f, tiny, std::ldexp(1.0f, -140), std::ldexp(1.0f, -126)}) {
            if (x <= amax) {
                bad += std::signbit(div.quotient(x)) || !std::signbit(div.quotient(-x));
                bad += std::signbit(kv::for_rounding(div.quotient(x))) || !std::signbit(kv::for_rounding(div.quotient(-x)));
            }
        }
    }
    return bad;
}

extern "C" {

uint64_t kv_check_signs(int format, int exponent, int wide)
{
    return wide != 0 ? check_signs<double>(format, exponent) : check_signs<float>(format, exponent);
}

uint64_t kv_check_int8(int bits, int max_gap, int exponent, uint64_t* slow)
{
    return bits > 8 ? check_int8<true>(bits, max_gap, exponent, slow) : check_int8<false>(bits, max_gap, exponent, slow);
}

// n / d by FastDiv against the machine's division for `count` values of n; the first that differs, or -1.
int64_t kv_check_fast_div(uint32_t d, const uint32_t* n, size_t count)
{
    const kv::FastDiv f = kv::make_fast_div(d);
    for (size_t i = 0; i < count; ++i) {
        if (kv::quotient(f, n[i]) != n[i] / d) {
            return static_cast<int64_t>(n[i]);
        }
    }
    return -1;
}

// vector_index of every vector of `objects` objects against nested loops; the number that differ.
uint64_t kv_check_vectors(uint32_t objects, uint32_t planes, uint32_t layers, uint32_t tokens, uint32_t heads)
{
    const uint32_t units = planes * layers * tokens * heads;
    const kv::FastDiv by_object = kv::make_fast_div(units), by_tokens = kv::make_fast_div(tokens);
    const kv::FastDiv by_layers = kv::make_fast_div(layers), by_heads = kv::make_fast_div(heads);
    uint64_t bad = 0;
    uint32_t v = 0;
    for (uint32_t o = 0; o < objects; ++o) {
        uint32_t in = 0;
        for (uint32_t p = 0; p < planes; ++p) {
            for (uint32_t l = 0; l < layers; ++l) {
                for (uint32_t t = 0; t < tokens; ++t) {
                    for (uint32_t h = 0; h < heads; ++h, ++v, ++in) {
                        const kv::VectorIndex x = kv::vector_index(v, by_object, by_tokens, by_layers, by_heads);
                        bad += x.object != o || x.in_object != in || x.plane != p || x.layer != l || x.token != t ||
                               x.head != h;
                    }
                }
            }
        }
    }
    return bad;
}

uint64_t kv_check_record_size(int format, uint32_t head_dim, uint64_t vectors)
{
    return kv::record_layout(format, head_dim, vectors).size;
}

uint64_t kv_check_quotients(int format, int bits, int max_gap, int step, int exponent)
{
    return bits > 11 ? check_quotients<double>(format, bits, max_gap, step, exponent)
                     : check_quotients<float>(format, bits, max_gap, step, exponent);
}

// scale_of against the machine's division for every float of a binade; the number that differ.
uint64_t kv_check_scales(int format, int exponent)
{
    uint64_t bad = 0;
    for (uint32_t m = 0; m < 1u << 23; ++m) {
        const float a = kv::bits_float(static_cast<uint32_t>(exponent + 127) << 23 | m);
        const float want = format == kv::kInt8 ? a / 127.0f : a / 448.0f;
        const float got = format == kv::kInt8 ? kv::scale_of<kv::kInt8>(a) : kv::scale_of<kv::kFp8>(a);
        bad += want != got;
    }
    return bad;
}

uint32_t kv_check_mx_byte(uint32_t bits) { return kv::mx_scale_byte(bits); }
float kv_check_mx_inverse(uint32_t byte) { return kv::mx_inverse(byte); }
float kv_check_scale(int format, float amax)
{
    return format == kv::kInt8 ? kv::scale_of<kv::kInt8>(amax) : kv::scale_of<kv::kFp8>(amax);
}

}  // extern "C"
