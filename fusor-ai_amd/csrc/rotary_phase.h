// The angles of rotary positions: position times frequency, in turns (plain C++: the kernels and the host share it).
#pragma once

#include <cmath>
#include <cstdint>

#include "cache_layout.h"

namespace fg {

// A pair's turn per token is kept as a fraction of 2^64, so that position * step, which drops whole turns as it
// overflows, is the fraction of the last one: off by position * 2^-65 turns for the step's rounding, at any position. (In
// f32 such a product has no digit left for far positions: past 2^20 radians its steps are 2^-3.)
//
// The angle of position p is that of the whole four positions before it and of p % 4 more tokens, together: four tokens in a row
// share the series, and a position's angle is the same to the bit wherever it is computed.
struct Angle {
    double c, s;
};
struct RotaryPair {
    uint64_t step;
    Angle more[4];  // by 0 to 3 tokens
};

// The cosine and sine of a phase: the nearest quarter turn is taken off exactly, and what is left, x in [-pi/4, pi/4], goes
// through Taylor's series, whose first dropped terms are x^17 / 17! < 5e-17 and x^18 / 18! < 3e-18.
FG_BOTH Angle angle_of(uint64_t phase)
{
    const uint64_t quarter = (phase + (uint64_t(1) << 61)) >> 62;
    const int64_t rest = int64_t(phase - (quarter << 62));
    const double x = double(rest) * 0x1.921fb54442d18p-62;  // 2 pi / 2^64
    const double y = x * x;
    double s = -1.0 / 1307674368000.0;
    s = __builtin_fma(s, y, 1.0 / 6227020800.0);
    s = __builtin_fma(s, y, -1.0 / 39916800.0);
    s = __builtin_fma(s, y, 1.0 / 362880.0);
    s = __builtin_fma(s, y, -1.0 / 5040.0);
    s = __builtin_fma(s, y, 1.0 / 120.0);
    s = __builtin_fma(s, y, -1.0 / 6.0);
    s = __builtin_fma(s * y, x, x);
    double c = 1.0 / 20922789888000.0;
    c = __builtin_fma(c, y, -1.0 / 87178291200.0);
    c = __builtin_fma(c, y, 1.0 / 479001600.0);
    c = __builtin_fma(c, y, -1.0 / 3628800.0);
    c = __builtin_fma(c, y, 1.0 / 40320.0);
    c = __builtin_fma(c, y, -1.0 / 720.0);
    c = __builtin_fma(c, y, 1.0 / 24.0);
    c = __builtin_fma(c, y, -0.5);
    c = __builtin_fma(c, y, 1.0);
    const bool odd = quarter & 1;
    Angle a;
    a.c = odd ? s : c;
    a.s = odd ? c : s;
    // quarters 1 and 2 have a negative cosine, 2 and 3 a negative sine
    if (((quarter + 1) & 2) != 0) a.c = -a.c;
    if ((quarter & 2) != 0) a.s = -a.s;
    return a;
}

FG_BOTH Angle both(const Angle &a, const Angle &b) { return Angle{__builtin_fma(a.c, b.c, -(a.s * b.s)), __builtin_fma(a.s, b.c, a.c * b.s)}; }
FG_BOTH Angle whole_four(const RotaryPair &r, int position) { return angle_of(uint64_t(unsigned(position) & ~3u) * r.step); }
FG_BOTH Angle angle_at(const RotaryPair &r, int position) { return both(whole_four(r, position), r.more[position & 3]); }

// `frequency` radians a token, of at most 1024 in magnitude, as a step: its turns' fraction, rounded to 2^-64, in whole numbers. The
// frequency's 53 bits times the first 126 of 1 / (2 pi) are off by less than 2^-53 of a step.
inline uint64_t turn_step(double frequency)
{
    constexpr uint64_t kHigh = 0x28be60db9391054a, kLow = 0x7f09d5f47d4d3770;  // 2^128 / (2 pi)
    int exponent;
    const uint64_t digits = uint64_t(std::ldexp(std::frexp(std::fabs(frequency), &exponent), 53));
    // digits 2^(exponent - 53) 2^64 / (2 pi), without the product's lowest 64 bits
    const unsigned __int128 product = (unsigned __int128)digits * kHigh + uint64_t(((unsigned __int128)digits * kLow) >> 64);
    const int drop = 53 - exponent;  // of its bits, at least 42
    uint64_t step = 0;
    if (drop <= 128) step = uint64_t(product >> (drop - 1) >> 1) + uint64_t(product >> (drop - 1) & 1);
    return frequency < 0 ? -step : step;
}

inline RotaryPair rotary_pair(double frequency)
{
    RotaryPair r;
    r.step = turn_step(frequency);
    for (uint64_t k = 0; k < 4; k++) r.more[k] = angle_of(k * r.step);
    return r;
}

}  // namespace fg
