// The weights that a draw adds up, w = exp((x - top) / T) in f64, and the order of scores.  Plain C++: the same code is
// inlined into the kernels (kernels_sample.hpp) and checked on the host (tests/test_vocabulary.py).
#pragma once

#include <math.h>
#include <stdint.h>

#if !defined(SERHIP_HD)
#if defined(__HIPCC__)
#define SERHIP_HD __host__ __device__ __forceinline__
#else
#define SERHIP_HD inline
#endif
#endif

namespace serhip {

template <typename To, typename From>
SERHIP_HD To bits_as(From x) {
    static_assert(sizeof(To) == sizeof(From), "the same bits");
    return __builtin_bit_cast(To, x);
}

// An unsigned number that orders like the score: 0 for -inf and NaN, -0 and +0 alike.
SERHIP_HD uint32_t score_key(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = bits_as<uint32_t>(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
SERHIP_HD float key_score(uint32_t k) { return bits_as<float>(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// 2^(j / kPowers), by the series of exp
constexpr int kPowers = 512;
struct PowerTable {
    double v[kPowers];
    constexpr PowerTable() : v{} {
        for (int j = 0; j < kPowers; ++j) {
            const double x = j * (0.6931471805599453 / kPowers);
            double sum = 1.0;
            for (int k = 24; k; --k) sum = 1.0 + sum * x / k;
            v[j] = sum;
        }
    }
};

constexpr float kLargestScore = 0x1.fffffep127f;
constexpr double kLog2E = 1.4426950408889634;

struct RowWeights {
    float top;        // the largest score
    float low;        // below it a score's weight is taken for that of `low`, 2^-200 or less (or `low` is the lowest number)
    float none;       // scores up to here have no weight: -inf, or every number where the largest score is +inf
    float ct;         // log2 e / T
    double top_wide;  // `top`; the largest number for +inf
    double ct_wide;   // kPowers log2 e / T
    double scale;     // 2^weight_bits
    // exp((x - top) / T) = 2^(n / kPowers) 2^(f / kPowers), |f| <= 1/2: the first factor from a table (power(j) =
    // 2^(j / kPowers)), the second by its series to the third power, 2^-46 of the result.  n is rounded, and read, as the
    // last bits of a sum with 2^52: 9 f64 instructions and one conversion, where a polynomial for |f| < 1/2 octave takes 14
    // and two.  They take two and four times the time of others (a row of 100 003 untruncated scores: 28 us with n from
    // f32, three instructions to keep x in range and a test of the result).  Exactly 1 at x = top.  Without branches, so that a
    // vector's weights are worked out together; for x > none only.  `low` keeps n above -1022 kPowers: the exponent that is
    // added to the table's would run into the sign.
    template <typename Power>
    SERHIP_HD double real(float x, Power power) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const float held = __builtin_amdgcn_fmed3f(x, low, kLargestScore);   // (NaN: low)
#else
        const float held = fminf(fmaxf(x, low), kLargestScore);
#endif
        const double d = static_cast<double>(held) - top_wide;
        const double sum = fma(d, ct_wide, 0x1.8p52), f = fma(d, ct_wide, 0x1.8p52 - sum);
        constexpr double c = 0.6931471805599453 / kPowers;
        const double g = fma(fma(fma(c * c * c / 6.0, f, c * c / 2.0), f, c), f, 1.0);
        const uint32_t n = static_cast<uint32_t>(bits_as<uint64_t>(sum));
        // n = kPowers times the exponent, and the rest: the exponent is added where an f64 has it
        const uint64_t first = bits_as<uint64_t>(static_cast<double>(power(n & (kPowers - 1))));
        const uint32_t high = static_cast<uint32_t>(first >> 32) + ((n & ~(kPowers - 1u)) << 11);
        return bits_as<double>(static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(first)) * g;
    }
    // round(w 2^bits), read off the mantissa of a sum with 2^52
    SERHIP_HD uint64_t whole(double w) const { return bits_as<uint64_t>(fma(w, scale, 0x1p52)) & ((1ull << 52) - 1); }
};
static_assert(kPowers == 1 << 9, "the exponent of n / kPowers");

// The weights of a row whose largest score is `top`, at temperature t >= 1e-30.
//
// `low` is `top` less 600 octaves, as an f32: it has to be off `top`, and not 1 022 octaves away from it.  Where an octave is
// small against the distance of f32 numbers at `top` (top = 10, t = 1e-9; top = 1e10, t = 1) it would round to `top` itself,
// and every class weigh 1, or to a number thousands of octaves down.  So an octave is never less than 1/400 of the distance
// from `top` to the next number below: the scores below weigh 2^-400 then, which is as nothing as what they should weigh.
// `low` is at least 1.5 of these distances down, and rounding moves it by at most one (the numbers lie twice as far
// apart past a power of two): by 400 octaves.
SERHIP_HD RowWeights row_weights(float top, float t, int bits) {
    const float held = fminf(top, kLargestScore);
    const double wide = static_cast<double>(held);
    const double gap = held > -kLargestScore ? wide - static_cast<double>(key_score(score_key(held) - 1)) : 0.0;
    const double least_t = gap * (kLog2E / 400.0);
    double held_t = t, ct_wide = kPowers * kLog2E / held_t;   // (a division that does not wait for `top`)
    if (held_t < least_t) {
        held_t = least_t;
        ct_wide = kPowers * kLog2E / held_t;
    }
    RowWeights rw;
    rw.top = top;
    rw.low = fmaxf(static_cast<float>(wide - held_t * (600.0 / kLog2E)), -kLargestScore);
    rw.none = top == INFINITY ? kLargestScore : -INFINITY;
    rw.ct = 1.44269504f / t;
    rw.top_wide = wide;
    rw.ct_wide = ct_wide;
    rw.scale = static_cast<double>(1ull << bits);
    return rw;
}

}  // namespace serhip
