// Quantising a block of 128 values to e4m3 under one fp32 scale, 16 lanes of 8 values each: shared by the row
// quantiser (nq_fp8_block.hip) and the layer norm that writes codes (nq_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nq {

template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}

// the largest of the 16 lanes of a DPP row, in every one of them
__device__ __forceinline__ uint32_t row16_umax(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));   // lane ^ 1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));   // lane ^ 2
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));  // the other quad of 8
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));  // the other half of 16
}

// s = amax / 448 (1 where the block is zero, never below 2^-126); q = e4m3(x / s), both divisions as IEEE rounds them,
// ties of the codes to even.  A block with a NaN or an infinity gets the scale NaN and codes 0x7F: all its values are
// NaN.  (A quotient beyond 448 is at most 448 (1 + 2^-23), which the conversion rounds to 448.)
// What bounds it is the vector ALU beside the stream, so nothing here is a division (a dozen instructions each).  A
// quotient a / b is q0 = RN(a r) with r = RN(1 / b), its exact remainder e = fma(q0, b, -a), and fma(-e, r, q0), which is
// RN(a / b) (Markstein, 1990); with the signs this way round a negative zero keeps its sign.  The remainder is exact
// while it is normal: a block of tiny values is lifted by 2^64 first, scale and values alike.  r itself is the
// hardware's reciprocal (within one unit in the last place) and one such step, which is RN(1 / b) unless b's
// significand is all ones.  Both exceptions are left to the wavefronts that meet one.  The maximum takes two values per
// instruction (v_maximum3_f32, which passes NaNs on) and crosses lanes as an integer, where a NaN is the largest.
__device__ __forceinline__ uint2 quantize_block16(const float (&x)[8], float& scale) {
    float v[8];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = x[i], most = __builtin_elementwise_maximum(most, __builtin_fabsf(x[i]));
    const uint32_t bits = row16_umax(__float_as_uint(most));
    const float top = __uint_as_float(bits);
    constexpr float R448 = 1.0f / 448.0f;
    const float s0 = top * R448;
    // (448 s0 - top is a multiple of 2^-143 wherever s >= 2^-126: exact)
    float s = fmaxf(fmaf(-fmaf(s0, 448.0f, -top), R448, s0), 0x1p-126f);
    if (bits == 0) s = 1.0f;
    const bool bad = bits >= 0x7F800000u;
    float sl = s;
    float r = __builtin_amdgcn_rcpf(s);
    r = fmaf(fmaf(-s, r, 1.0f), r, r);
    if (__any(s < 0x1p-60f || (__float_as_uint(s) & 0x007FFFFFu) == 0x007FFFFFu)) {
        const float lift = s < 0x1p-60f ? 0x1p64f : 1.0f;
        sl *= lift;
        r = 1.0f / sl;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= lift;
    }
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float q0 = v[i] * r;
        const float e = fmaf(q0, sl, -v[i]);
        q[i] = fmaf(-e, r, q0);
    }
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    scale = bad ? __uint_as_float(0x7FC00000u) : s;
    return bad ? make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu) : make_uint2((uint32_t)lo, (uint32_t)hi);
}

}  // namespace nq
