// Quantising a block of 128 values to e4m3 under one fp32 scale, 16 lanes of 8 values each: shared by the row
// quantiser (nq_fp8_block.hip) and the layer norm that writes codes (nq_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nq {

// the largest of the 16 lanes of a DPP row, in every one of them
__device__ __forceinline__ uint32_t row16_umax(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, false));  // row_ror:1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false));
    return v;
}

// s = amax / 448 (1 where the block is zero, never below 2^-126); q = e4m3(clip(x / s)), both divisions as IEEE
// rounds them, ties of the codes to even.  A block with a NaN or an infinity gets the scale NaN and codes 0x7F: all its
// values are NaN.  (Magnitudes are compared as integers, where every NaN is larger than infinity.)
// The quotients are not divisions: with r = RN(1 / s), q0 = RN(x r) and the exact remainder e = fma(q0, s, -x),
// fma(-e, r, q0) is RN(x / s) (Markstein, 1990), three instructions instead of a dozen; with the signs this way round a
// negative zero keeps its sign.  The remainder is exact while it is normal, so a block of tiny values is lifted by 2^64
// first, scale and values alike.
__device__ __forceinline__ uint2 quantize_block16(const float (&v)[8], float& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = row16_umax(top);
    float s = fmaxf(__uint_as_float(top) / 448.0f, 0x1p-126f);
    if (top == 0) s = 1.0f;
    const bool bad = top >= 0x7F800000u;
    const float lift = s < 0x1p-60f ? 0x1p64f : 1.0f;
    const float sl = s * lift, r = 1.0f / sl;
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = v[i] * lift;
        const float q0 = t * r;
        const float e = fmaf(q0, sl, -t);
        q[i] = __builtin_amdgcn_fmed3f(fmaf(-e, r, q0), -448.0f, 448.0f);
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
