// Groups of 32 values as e4m3 codes with one power of two (e8m0): what add_norm.hip and rope_kv.hip write, linear_w4.hip and attention_decode.hip read.
#pragma once
#include "common.h"

namespace moe {

MOE_DEVICE uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Maximum over groups of LANES (8, 32 or 64) neighbouring lanes, in all of them.
template <int LANES>
MOE_DEVICE uint32_t group_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));   // lanes that differ in bit 0,
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));   // bit 1,
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));  // mirrored in 8 lanes,
    if constexpr (LANES > 8) {
        v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));  // in 16,
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);             // neighbouring rows,
        v = max(r[0], r[1]);
    }
    if constexpr (LANES > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);  // halves
        v = max(r[0], r[1]);
    }
    return v;
}

// Power-of-two scale of a group (e8m0): the smallest 2^(b - 127), b >= 1, that brings its largest value to 448 or below.  448 = 1.75 * 2^8, so
// the exponent field goes up by one where the mantissa is past 1.75.  255 where the group holds an infinity or a NaN.
MOE_DEVICE uint32_t mx_scale_byte(uint32_t amax) {
    if (amax >= 0x7F800000u) return 255u;
    const int b = (int)((amax + 0x1FFFFFu) >> 23) - 8;
    return (uint32_t)max(b, 1);
}

// v in fp32 with the bits that there is no room for gathered in the last one (odd if anything was cut off), so that the rounding to fewer bits that follows is
// the only one: a value next to the middle of two codes does not become it.
MOE_DEVICE float to_odd(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)b;
    const uint32_t odd = min(lo & 0x1FFFFFFFu, 1u) << 29;
    return (float)__builtin_bit_cast(double, (b & 0xFFFFFFFFE0000000ull) | odd);
}

// e4m3 values times a power of two (its exponent counts: the bits of 0 are 2^-127), to bf16: exact, with three mantissa bits, but for denormals.
MOE_DEVICE u32x4 e4m3x8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
    u32x4 v;
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return v;
}

}  // namespace moe
