// Rotary positions: the angle of a (position, pair), in 64 bits.
//
// A pair (a, b) at position p turns by the angle p f of its frequency f: (a cos - b sin, b cos + a sin).  Frequencies are float64 and the
// angle is never rounded to fewer bits: in float32 the angle of position 100000 is off by up to 0.004 radians, in float64 by 1e-11.  Only the
// cosine and sine, times the amplitude, are rounded to float32, once.
#pragma once

#include "terna_common.h"

namespace terna {

// sin and cos of r, |r| <= pi / 4 (and a little): their Taylor series up to r^17 and r^16, whose next terms are below 2^-58.
__device__ __forceinline__ double rotary_sin(double r, double r2)
{
    double p = 1.0 / 355687428096000.0;                                  // 1 / 17!
    p = fma(p, r2, -1.0 / 1307674368000.0);
    p = fma(p, r2, 1.0 / 6227020800.0);
    p = fma(p, r2, -1.0 / 39916800.0);
    p = fma(p, r2, 1.0 / 362880.0);
    p = fma(p, r2, -1.0 / 5040.0);
    p = fma(p, r2, 1.0 / 120.0);
    p = fma(p, r2, -1.0 / 6.0);
    return fma(p * r2, r, r);
}
__device__ __forceinline__ double rotary_cos(double r2)
{
    double p = 1.0 / 20922789888000.0;                                   // 1 / 16!
    p = fma(p, r2, -1.0 / 87178291200.0);
    p = fma(p, r2, 1.0 / 479001600.0);
    p = fma(p, r2, -1.0 / 3628800.0);
    p = fma(p, r2, 1.0 / 40320.0);
    p = fma(p, r2, -1.0 / 720.0);
    p = fma(p, r2, 1.0 / 24.0);
    p = fma(p, r2, -0.5);
    return fma(p, r2, 1.0);
}

// (cos, sin) of position * frequency, times the amplitude.  The angle loses its quarter turns by two fused steps: pi / 2 in two parts, whose
// product with the number of quarter turns is exact inside the fused operation.
__device__ __forceinline__ float2 rotary_angle(long long position, double frequency, double amplitude)
{
    constexpr double kHalfPi = 1.5707963267948966, kHalfPiRest = 6.123233995736766e-17;
    const double angle = static_cast<double>(position) * frequency;
    const double turns = rint(angle * 0.6366197723675814);               // 2 / pi
    const double r = fma(-turns, kHalfPiRest, fma(-turns, kHalfPi, angle));
    const double r2 = r * r;
    const double s = rotary_sin(r, r2), c = rotary_cos(r2);
    const int quarter = static_cast<int>(static_cast<long long>(turns)) & 3;
    double cs = quarter & 1 ? s : c, sn = quarter & 1 ? c : s;
    if (quarter == 1 || quarter == 2) cs = -cs;
    if (quarter >= 2) sn = -sn;
    return float2{static_cast<float>(cs * amplitude), static_cast<float>(sn * amplitude)};
}

// The turned pair, every product and sum rounded by itself (the same bits wherever a row is turned).
__device__ __forceinline__ float2 rotary_turn(float a, float b, float2 cs)
{
#pragma clang fp contract(off)
    return float2{a * cs.x - b * cs.y, b * cs.x + a * cs.y};
}

}  // namespace terna
