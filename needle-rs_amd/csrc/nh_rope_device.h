// Cosine and sine of a position's angle, and a pair's rotation.
#pragma once

#include "nh_device.h"
#include "nh_rope.h"

namespace nh {

// amplitude cos and amplitude sin of position * frequency, rounded to f32.
//
// The frequency is held as turns a position in fractions of 2^64, so the
// product with a position modulo 2^64 is the angle modulo a whole turn: exact at
// any position, where an f32 product is off by a radian at 10^7.  The nearest
// quarter turn is taken off, and the rest |x| <= pi/4 goes into the two Taylor
// series to x^13 and x^14 in f64 (the first terms left out are below 2^-45 and
// 2^-49), which round to f32 as the exact values do but for one in about 2^20.
// f64 runs at f32's rate here; both cost about 40 instructions.
__device__ __forceinline__ float2 rope_cos_sin(uint64_t turns, int pos, double amplitude) {
    const uint64_t t = (uint64_t)(int64_t)pos * turns;
    const uint32_t quarter = (uint32_t)((t + (1ull << 61)) >> 62);
    const int64_t rest = (int64_t)(t - ((uint64_t)quarter << 62));
    const double x = (double)rest * 3.4061215800865545e-19;  // 2 pi / 2^64
    const double z = x * x;
    double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    s = __builtin_fma(s * z, x, x);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const bool odd = quarter & 1;
    const double a = odd ? s : c, b = odd ? c : s;
    const float co = (float)(amplitude * a), si = (float)(amplitude * b);
    // quarters 0 .. 3: (c, s), (-s, c), (-c, -s), (s, -c)
    return float2{(quarter + 1) & 2 ? -co : co, quarter & 2 ? -si : si};
}

// (a, b) turned by (c, s): each product and sum rounded to f32 of its own, so
// that a turned key is the same number wherever it is turned.
__device__ __forceinline__ float2 rope_turn(float a, float b, float2 cs) {
    return float2{a * cs.x - b * cs.y, b * cs.x + a * cs.y};
}

}  // namespace nh
