// kv8_core.h - the e4m3 arithmetic of the 8-bit KV cache (kv_layout.h: blocks
// of e4m3 bytes with a power-of-two fp32 scale per plane), shared by the
// append and the decode attention.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_layout.h"
#include "rl_dev_common.h"

namespace {

// The biased exponent of the smallest power of two s with amax <= 448 s, not
// below 2^-126 (amax finite and not negative): amax = m 2^e reaches 1.75 2^8 s.
// With 1 <= exponent <= 247, s and 1 / s are both normal numbers.
__device__ __forceinline__ uint32_t kv8_scale_exponent(float amax)
{
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(e, 1);
}
__device__ __forceinline__ float kv8_scale(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ float kv8_inverse(uint32_t exponent) { return __uint_as_float((254u - exponent) << 23); }

// Four floats of magnitude at most 448 (or NaN) -> four e4m3 bytes, nearest even.
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Two e4m3 bytes (the low or high half of w) -> two packed 16-bit values,
// exactly: unscaled as bf16 or fp16 ...
template <int DT, bool HIGH>
__device__ __forceinline__ uint32_t kv8_unpack2(uint32_t w)
{
    if constexpr (DT == 0)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
}
// ... or times a power of two as bf16.
template <bool HIGH>
__device__ __forceinline__ uint32_t kv8_unpack2_scaled(uint32_t w, float scale)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}

// 4 x 4 bytes transposed: out[j] holds byte j of rows 0 .. 3.
__device__ __forceinline__ void kv8_transpose4(const uint32_t (&r)[4], uint32_t (&out)[4])
{
    // __builtin_amdgcn_perm(a, b, sel): selector values 0-3 pick bytes of b, 4-7 bytes of a
    const uint32_t p01l = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u);  // r0.0 r1.0 r0.1 r1.1
    const uint32_t p01h = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);  // r0.2 r1.2 r0.3 r1.3
    const uint32_t p23l = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u);
    const uint32_t p23h = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(p23l, p01l, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(p23l, p01l, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(p23h, p01h, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(p23h, p01h, 0x07060302u);
}

}  // namespace
