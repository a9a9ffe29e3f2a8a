// Shared by the block-scaled fp8 product's kernels (nq_fp8_block.hip: few rows; nq_fp8_block_gemm.hip: many).
#pragma once

#include <type_traits>

#include "nq_common.h"

namespace nq {

// f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, I + 1>(static_cast<F&&>(f));
    }
}

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

// A lane's 32 bytes of an operand (16 rows x 128 k): as they are, or decoded to bf16 in four operands of 32 k each.
// (A lane's k within an operand are the same 8 for both sides; which 8 they are does not matter to a sum.)
template <bool EXACT>
struct Operand;
template <>
struct Operand<false> {
    i32x8 v;
    __device__ Operand() {}
    __device__ __forceinline__ Operand(const i32x4& a, const i32x4& b) : v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]} {}
};
template <>
struct Operand<true> {
    bf16x8 v[4];
    __device__ Operand() {}
    __device__ __forceinline__ Operand(const i32x4& a, const i32x4& b) {
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int w = s < 2 ? a[2 * s + h] : b[2 * (s - 2) + h];
                const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
                const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
                v[s][4 * h] = lo[0], v[s][4 * h + 1] = lo[1], v[s][4 * h + 2] = hi[0], v[s][4 * h + 3] = hi[1];
            }
    }
};

// one block's sums: 16 weight rows (result rows) x 16 activation rows (result columns)
__device__ __forceinline__ f32x4 block_sum(const Operand<false>& w, const Operand<false>& x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f32x4{}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 block_sum(const Operand<true>& w, const Operand<true>& x) {
    f32x4 d = {};
#pragma unroll
    for (int s = 0; s < 4; s++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[s], x.v[s], d, 0, 0, 0);
    return d;
}

struct BlockParams {
    const uint8_t* x;   // codes [M][K]
    const uint8_t* w;   // tiles [ceil(N / 16)][G][2 KiB]
    const float* xs;    // [M][G]
    const float* ws;    // [ceil(N / 128)][G]
    const void* bias;
    int32_t M, N, K, G;
    int32_t tiles_m, tiles_n;
    int32_t m_base, n_base;  // the GEMM: its tiles count from here
    int32_t y_dtype, bias_dtype, relu;
    int32_t vec;  // the few-rows kernel: y can be written four channels at a time
    SegTable seg;
};

// nq_fp8_block_gemm.hip: whether the GEMM takes the call, and the time it is expected to take
bool fp8_block_gemm_estimate_us(const BlockParams& p, double* us);
void fp8_block_gemm_form(const BlockParams& p, int32_t* form);  // of a call that it takes: nq_diag_fp8_block_form
int32_t launch_fp8_block_gemm(const BlockParams& p, hipStream_t s);

}  // namespace nq
