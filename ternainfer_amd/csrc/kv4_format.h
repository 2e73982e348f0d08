// The 4-bit key/value cache: a row of D dimensions as D / 2 bytes of codes and D / 32 scale bytes.
//
// A code is e2m1 -- 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign, two to a byte, the even dimension in the lower half -- and stands for code times
// 2^(byte - 127) of its 32 dimensions' scale byte.  The exponent of 32 values is the smallest e with max |x| <= 7 * 2^e, so that the largest loses at
// most one unit (6 is nearest to 7 too: no worse than the half step between 4 and 6), held to -125 .. 125: every value is then a normal bf16
// number.  Codes round to nearest, ties to even, and end at 6.  Scale byte 255: one of the 32 values was NaN or infinite, and all stand for NaN.
// 4.25 bits a value.  gfx950 converts both ways in hardware, two values an instruction, the scale among its operands (checked for every code and scale and
// for values on and next to every border between codes: the conversions are these rules, and an exponent byte of 255 gives NaN).
#pragma once

#include "terna_common.h"

namespace terna {

constexpr int kKv4Group = 32;                  // dimensions that share a scale byte
constexpr uint32_t kKv4Broken = 255;           // its values stand for NaN
constexpr uint32_t kKv4MaxByte = 252;          // 2^125: the largest that is written beside it

// Scale byte of 32 values from the bits of their largest magnitude.
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t amax_bits)
{
    // 2^k * m <= 7 * 2^e with 1 <= m < 2: e = k - 2 up to m = 1.75, else k - 1
    const int byte = static_cast<int>((amax_bits + 0x1fffffu) >> 23) - 2;
    return amax_bits >= 0x7f800000u ? kKv4Broken : static_cast<uint32_t>(min(max(byte, 2), static_cast<int>(kKv4MaxByte)));
}

// Eight values -> eight codes.
__device__ __forceinline__ uint32_t kv4_codes(const float x[8], uint32_t byte)
{
    const float scale = __uint_as_float(byte << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
    return byte == kKv4Broken ? 0u : c;
}

// Eight codes -> eight bf16.
__device__ __forceinline__ u32x4 kv4_values(uint32_t codes, float scale)
{
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

}  // namespace terna
