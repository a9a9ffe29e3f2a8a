// Layer norm over rows of D values, and its gradient:
//     mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) rstd gamma + beta
//     a = gy gamma, xh = (x - mean) rstd:  gx = rstd (a - mean(a) - xh mean(a xh)),
//     dgamma = sum_m gy xh, dbeta = sum_m gy
// y leaves as fp32, bf16, or as the e4m3 codes and scales of blocks of 128 that an FP8_BLOCK layer reads.  Statistics and
// sums are fp32; the variance is summed from the centred values.
#include "nq_common.h"
#include "nq_fp8_quant.h"

namespace nq {

namespace {

__device__ __forceinline__ float load1(const void* p, int32_t dtype, int64_t i) {
    return dtype == NQ_DT_F32 ? reinterpret_cast<const float*>(p)[i]
                              : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}

__device__ __forceinline__ void store1(void* p, int32_t dtype, int64_t i, float v) {
    if (dtype == NQ_DT_F32) {
        reinterpret_cast<float*>(p)[i] = v;
    } else {
        uint32_t b = __float_as_uint(v);
        b = (b & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC0u : (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
        reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)b;
    }
}

// sum over a workgroup of 256, the same bits in every thread
__device__ __forceinline__ float block_sum(float v, float* lds) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// one workgroup per row
__global__ __launch_bounds__(256) void layer_norm_kernel(const NormArgs a) {
    __shared__ float lds[4];
    const int64_t m = blockIdx.x, base = m * a.D;
    float sum = 0.0f;
    for (int d = threadIdx.x; d < a.D; d += 256) sum += load1(a.x, a.x_dtype, base + d);
    const float mean = block_sum(sum, lds) / (float)a.D;
    float sq = 0.0f;
    for (int d = threadIdx.x; d < a.D; d += 256) {
        const float t = load1(a.x, a.x_dtype, base + d) - mean;
        sq += t * t;
    }
    const float rstd = 1.0f / sqrtf(block_sum(sq, lds) / (float)a.D + a.eps);
    if (threadIdx.x == 0 && a.mean) a.mean[m] = mean, a.rstd[m] = rstd;
    for (int d0 = 0; d0 < a.D; d0 += 2048) {
        const int d1 = d0 + 8 * (int)threadIdx.x;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = d1 + i;
            v[i] = 0.0f;
            if (d < a.D)
                v[i] = (load1(a.x, a.x_dtype, base + d) - mean) * rstd * (a.gamma ? a.gamma[d] : 1.0f) + (a.beta ? a.beta[d] : 0.0f);
        }
        if (a.y) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (d1 + i < a.D) store1(a.y, a.y_dtype, base + d1 + i, v[i]);
        } else {
            float s;
            const uint2 q = quantize_block16(v, s);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (d1 + i < a.D) a.codes[base + d1 + i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
            if ((threadIdx.x & 15) == 0 && d1 < a.D) a.scales[m * ((a.D - 1) / 128 + 1) + d1 / 128] = s;
        }
    }
}

// one workgroup per row
__global__ __launch_bounds__(256) void layer_norm_grad_x_kernel(const NormGradArgs a) {
    __shared__ float lds[4];
    const int64_t m = blockIdx.x, base = m * a.D;
    const float mean = a.mean[m], rstd = a.rstd[m];
    float s1 = 0.0f, s2 = 0.0f;
    for (int d = threadIdx.x; d < a.D; d += 256) {
        const float t = load1(a.gy, a.gy_dtype, base + d) * (a.gamma ? a.gamma[d] : 1.0f);
        s1 += t;
        s2 += t * ((load1(a.x, a.x_dtype, base + d) - mean) * rstd);
    }
    const float c1 = block_sum(s1, lds) / (float)a.D, c2 = block_sum(s2, lds) / (float)a.D;
    for (int d = threadIdx.x; d < a.D; d += 256) {
        const float t = load1(a.gy, a.gy_dtype, base + d) * (a.gamma ? a.gamma[d] : 1.0f);
        const float xh = (load1(a.x, a.x_dtype, base + d) - mean) * rstd;
        store1(a.gx, a.gx_dtype, base + d, rstd * (t - c1 - xh * c2));
    }
}

// one thread per column
__global__ __launch_bounds__(64) void layer_norm_grad_w_kernel(const NormGradArgs a) {
    const int d = blockIdx.x * 64 + threadIdx.x;
    if (d >= a.D) return;
    float g = 0.0f, b = 0.0f;
    for (int64_t m = 0; m < a.M; m++) {
        const float t = load1(a.gy, a.gy_dtype, m * a.D + d);
        g += t * ((load1(a.x, a.x_dtype, m * a.D + d) - a.mean[m]) * a.rstd[m]);
        b += t;
    }
    a.dgamma[d] = g, a.dbeta[d] = b;
}

}  // namespace

int32_t launch_layer_norm(const NormArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(layer_norm_kernel, dim3((unsigned)a.M), dim3(256), 0, s, a);
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

int64_t layer_norm_grad_partial_bytes(int32_t M, int32_t D) {
    (void)M, (void)D;
    return 0;
}

int32_t launch_layer_norm_grad(const NormGradArgs& a, hipStream_t s) {
    // (the columns first: gx may be gy's own memory)
    if (a.dgamma) {
        hipLaunchKernelGGL(layer_norm_grad_w_kernel, dim3((unsigned)((a.D + 63) / 64)), dim3(64), 0, s, a);
        NQ_HIP(hipGetLastError());
    }
    if (a.M) {
        hipLaunchKernelGGL(layer_norm_grad_x_kernel, dim3((unsigned)a.M), dim3(256), 0, s, a);
        NQ_HIP(hipGetLastError());
    }
    return NQ_OK;
}

}  // namespace nq
