// Layer norm over rows of D values, and its gradient:
//     mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) rstd gamma + beta
//     a = gy gamma, xh = (x - mean) rstd:  gx = rstd (a - mean(a) - xh mean(a xh)),
//     dgamma = sum_m gy xh, dbeta = sum_m gy
// y leaves as fp32, bf16, or as the e4m3 codes and scales of blocks of 128 that an FP8_BLOCK layer reads.  Statistics and
// sums are fp32; the variance is summed from the centred values.
//
// Bound by memory: each row is read once (backward: x and gy) and each result written once.  A team of T threads
// owns a row at a time and holds it in registers, 8 values per thread and vector, so the second pass over the centred
// values costs no memory; gamma and beta are read once per team and kept while it walks its rows, and the next row is
// requested before the current one is reduced.  T grows with D (64 threads up to 1024 values, where no barrier is needed;
// 256 up to 4096, 512 up to 8192, 1024 up to 16384) so that a thread holds at most 16 values of a row; longer rows are
// walked in passes (the *_long kernels).
// Measured, 8192 x 4096 in bf16: y in bf16 24 us (134 MB, 5.6 TB/s, a copy's rate), codes 22.5 - 23.3 (102 MB, 4.4 TB/s: the
// vector ALU, about 13 instructions a value, beside the two barriers a row); backward 38.3 + 4.8 (201 MB, 5.2 TB/s, and the
// partials).  fp32 in and out: 42 - 46 us (5.9 - 6.4 TB/s).
//
// 16 lanes hold 128 adjacent values: the block that shares a scale, so the quantised form needs one reduction over a DPP
// row per vector and nothing else.  Rows whose length is no multiple of 8 are not 16-byte aligned: there a lane takes
// every 16th value of its block instead of 8 adjacent ones, one load each (8192 x 4095 in bf16: 32 - 35 us).
#include <algorithm>

#include "nq_common.h"
#include "nq_fp8_quant.h"

namespace nq {

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

__device__ __forceinline__ float load1(const void* p, int32_t dtype, int64_t i) {
    return dtype == NQ_DT_F32 ? reinterpret_cast<const float*>(p)[i]
                              : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}

__device__ __forceinline__ void store1(void* p, int32_t dtype, int64_t i, float v) {
    if (dtype == NQ_DT_F32)
        reinterpret_cast<float*>(p)[i] = v;
    else
        reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
}

// sum over a wavefront, the same bits in every lane: neighbours, pairs, halves and rows of 16 by exchanges in which both
// sides add the same two numbers, then the four rows
__device__ __forceinline__ float wave_sum(float v) {
    v += lane_move<0xB1>(v);   // lane ^ 1
    v += lane_move<0x4E>(v);   // lane ^ 2
    v += lane_move<0x141>(v);  // the other quad of 8
    v += lane_move<0x140>(v);  // the other half of 16
    const int i = __float_as_int(v);
    return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
           (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

// sum over a team of T threads; `at`: this reduction's own T / 64 floats of LDS.  One barrier: two reductions that
// follow each other use different places, and the barrier of the one proves that the other has been read.
template <int T>
__device__ __forceinline__ float team_sum(float v, float* at, int wave_in_team) {
    v = wave_sum(v);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) at[wave_in_team] = v;
        __syncthreads();
        v = at[0];
#pragma unroll
        for (int w = 1; w < T / 64; w++) v += at[w];
    }
    return v;
}

// ---- a thread's 8 values of a vector: raw as loaded (so that a request can stay under way), then as fp32
template <bool BF16>
struct Raw {
    u32x4 v[BF16 ? 1 : 2];
};
// VEC: from index k on; otherwise every 16th value from k on.  Indices from `end` on give zeros and are not read.
template <bool BF16, bool VEC>
__device__ __forceinline__ void fetch(Raw<BF16>& r, const void* row, int k, int end) {
    if constexpr (VEC) {
#pragma unroll
        for (int h = 0; h < (BF16 ? 1 : 2); h++) r.v[h] = u32x4{0, 0, 0, 0};
        if (k < end) {  // (end is a multiple of 8)
            const u32x4* p = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(row) + (int64_t)k * (BF16 ? 2 : 4));
#pragma unroll
            for (int h = 0; h < (BF16 ? 1 : 2); h++) r.v[h] = p[h];
        }
    } else {
        // (loads without a branch each, behind which the compiler waits for every one: the row's last value again beyond its end)
        uint32_t t[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (end > 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int at = min(k + 16 * i, end - 1);
                const uint32_t v = BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(row)[at] : reinterpret_cast<const uint32_t*>(row)[at];
                t[i] = k + 16 * i < end ? v : 0;
            }
        }
        if constexpr (BF16) {
            r.v[0] = u32x4{t[0] | t[1] << 16, t[2] | t[3] << 16, t[4] | t[5] << 16, t[6] | t[7] << 16};
        } else {
            r.v[0] = u32x4{t[0], t[1], t[2], t[3]}, r.v[1] = u32x4{t[4], t[5], t[6], t[7]};
        }
    }
}
template <bool BF16>
__device__ __forceinline__ void widen(const Raw<BF16>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            f[2 * i] = __uint_as_float(r.v[0][i] << 16), f[2 * i + 1] = __uint_as_float(r.v[0][i] & 0xFFFF0000u);
        } else {
            f[i] = __uint_as_float(r.v[0][i]), f[4 + i] = __uint_as_float(r.v[1][i]);
        }
    }
}
template <bool VEC>
__device__ __forceinline__ void put(void* out, int32_t dtype, int64_t base, int k, int end, const float (&f)[8]) {
    if constexpr (VEC) {
        if (k >= end) return;
        if (dtype == NQ_DT_F32) {
            f32x4* p = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(out) + base + k);
            p[0] = f32x4{f[0], f[1], f[2], f[3]}, p[1] = f32x4{f[4], f[5], f[6], f[7]};
        } else {
            *reinterpret_cast<bf16x8*>(reinterpret_cast<uint16_t*>(out) + base + k) =
                __builtin_convertvector((f32x8{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]}), bf16x8);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (k + 16 * i < end) store1(out, dtype, base + k + 16 * i, f[i]);
    }
}
// the first index of thread t's vector v
template <int T, bool VEC>
__device__ __forceinline__ int first_index(int t, int v) {
    return VEC ? (v * T + t) * 8 : (v * T / 16 + t / 16) * 128 + t % 16;
}

// ---- forward: a workgroup of max(T, 256) threads, 256 / T teams of their own rows (T = 64: one wavefront each)
template <int T, int NV, bool BF16, bool VEC>
__global__ __launch_bounds__(T < 256 ? 256 : T) void layer_norm_kernel(const NormArgs a, int32_t teams) {
    __shared__ float lds[2][T / 64];
    constexpr int PER = T < 256 ? 256 / T : 1;
    const int t = threadIdx.x % T, team = (int)blockIdx.x * PER + (int)threadIdx.x / T;
    const int wave = t / 64;
    const int xs = BF16 ? 2 : 4;
    const float d = (float)a.D;
    const int blocks = (a.D - 1) / 128 + 1;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x);
    int64_t m = team;
    if (m >= a.M) return;  // (T >= 256: a team is a workgroup, so a workgroup's threads leave together)
    Raw<BF16> cur[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) fetch<BF16, VEC>(cur[v], x + m * a.D * xs, first_index<T, VEC>(t, v), a.D);
    float g[NV][8], b[NV][8];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int k = first_index<T, VEC>(t, v);
        Raw<false> r;
        // (a thread's values behind the row get zeros here, so that they come out as zeros: what the last block's largest
        // magnitude may not see)
#pragma unroll
        for (int i = 0; i < 8; i++) g[v][i] = (VEC ? k : k + 16 * i) < a.D ? 1.0f : 0.0f, b[v][i] = 0.0f;
        if (a.gamma) fetch<false, VEC>(r, a.gamma, k, a.D), widen<false>(r, g[v]);
        if (a.beta) fetch<false, VEC>(r, a.beta, k, a.D), widen<false>(r, b[v]);
    }
    for (;;) {
        const int64_t next = m + teams;
        float f[NV][8];
#pragma unroll
        for (int v = 0; v < NV; v++) widen<BF16>(cur[v], f[v]);
        if (next < a.M) {
#pragma unroll
            for (int v = 0; v < NV; v++) fetch<BF16, VEC>(cur[v], x + next * a.D * xs, first_index<T, VEC>(t, v), a.D);
        }
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int i = 0; i < 8; i++) sum += f[v][i];
        const float mean = team_sum<T>(sum, lds[0], wave) / d;
        float sq = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int k = first_index<T, VEC>(t, v);
            const float centre = !VEC || k < a.D ? mean : 0.0f;
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // (zeros behind the row stay zeros: a mean beyond 2^128 / rstd would make them infinite below, and those a
                // NaN in the last block's largest magnitude)
                f[v][i] = VEC || k + 16 * i < a.D ? f[v][i] - centre : 0.0f;
                part = VEC ? fmaf(f[v][i], f[v][i], part) : part + f[v][i] * f[v][i];
            }
            sq += part;
        }
        const float rstd = 1.0f / sqrtf(team_sum<T>(sq, lds[1], wave) / d + a.eps);
        if (a.mean && t == 0) a.mean[m] = mean, a.rstd[m] = rstd;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int k = first_index<T, VEC>(t, v);
#pragma unroll
            for (int i = 0; i < 8; i++) f[v][i] = f[v][i] * rstd * g[v][i] + b[v][i];
            if (a.y) {
                put<VEC>(a.y, a.y_dtype, m * a.D, k, a.D, f[v]);
            } else {
                float s;
                const uint2 q = quantize_block16(f[v], s);
                if constexpr (VEC) {
                    if (k < a.D) *reinterpret_cast<uint2*>(a.codes + m * a.D + k) = q;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (k + 16 * i < a.D) a.codes[m * a.D + k + 16 * i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
                }
                if (t % 16 == 0 && k < a.D) a.scales[m * blocks + (v * T + t) / 16] = s;
            }
        }
        if (next >= a.M) break;
        m = next;
    }
}

// Rows beyond 16384 values: one workgroup per row, three passes (the row comes from the caches after the first), one value per
// load.  1024 x 32768: 157 us in fp32 (1.7 TB/s), 125 in bf16 (1.1), 145 and 123 into codes; the gradient below 174 and 177.
// Half the bytes take nearly the same time: the number of loads bounds it, not memory (54 and 27 us; 81 and 40).
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(const NormArgs a) {
    __shared__ float lds[2][16];
    const int wave = threadIdx.x / 64;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const int64_t base = m * a.D;
        float sum = 0.0f;
        for (int64_t d = threadIdx.x; d < a.D; d += 1024) sum += load1(a.x, a.x_dtype, base + d);
        const float mean = team_sum<1024>(sum, lds[0], wave) / (float)a.D;
        float sq = 0.0f;
        for (int64_t d = threadIdx.x; d < a.D; d += 1024) {
            const float t = load1(a.x, a.x_dtype, base + d) - mean;
            sq += t * t;
        }
        const float rstd = 1.0f / sqrtf(team_sum<1024>(sq, lds[1], wave) / (float)a.D + a.eps);
        if (threadIdx.x == 0 && a.mean) a.mean[m] = mean, a.rstd[m] = rstd;
        for (int64_t d0 = 0; d0 < a.D; d0 += 8192) {
            const int64_t k = d0 + (int64_t)(threadIdx.x / 16) * 128 + threadIdx.x % 16;  // every 16th value of a block
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int64_t d = k + 16 * i;
                f[i] = 0.0f;
                if (d < a.D) f[i] = (load1(a.x, a.x_dtype, base + d) - mean) * rstd * (a.gamma ? a.gamma[d] : 1.0f) + (a.beta ? a.beta[d] : 0.0f);
            }
            if (a.y) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (k + 16 * i < a.D) store1(a.y, a.y_dtype, base + k + 16 * i, f[i]);
            } else {
                float s;
                const uint2 q = quantize_block16(f, s);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (k + 16 * i < a.D) a.codes[base + k + 16 * i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
                if (threadIdx.x % 16 == 0 && k < a.D) a.scales[m * ((a.D - 1) / 128 + 1) + k / 128] = s;
            }
        }
    }
}

// ---- backward.  A workgroup is 1024 threads = 1024 / T teams; each team adds its rows' gy xh and gy into registers,
// the teams' sums meet in LDS in team order, and a workgroup writes ONE partial of dgamma | dbeta, so that at most 256
// partials (one workgroup per CU) are left to add: 2 D fp32 each, 8 MB for D = 4096 against 200 of rows at M = 8192.
// A thread holds 8 values of x, gy, gamma and both sums and the next row's raw 8 (90 registers of the 128 that 16
// wavefronts per CU leave it); with 16 of each it spilled (8192 x 4096 in bf16: 76 us a call against 40).  Rows of more than
// 8192 values have 16 per thread and do without the early request (AHEAD), and still put a few of them in scratch memory:
// 12 - 20 bytes per lane, 84 where the length is no multiple of 8 (noeira_amd/build.py holds them to that).  8192 x 11008
// takes 133 us in bf16 (4.1 TB/s) and 219 in fp32 (4.9), 2048 x 16384 66 and 105.
template <int T, int NV, bool XB, bool GB, bool VEC>
__global__ __launch_bounds__(1024) void layer_norm_grad_kernel(const NormGradArgs a, int32_t rounds) {
    extern __shared__ __attribute__((aligned(16))) float meet[];  // [2][T * 8 * NV] where there are teams to meet
    __shared__ float lds[2][1024 / T][2][T / 64];
    constexpr int TEAMS = 1024 / T, W = T * 8 * NV;
    constexpr bool AHEAD = NV == 1;
    const int t = threadIdx.x % T, mine = (int)threadIdx.x / T;
    const int wave = t / 64;
    const int64_t teams = (int64_t)gridDim.x * TEAMS;
    const float inv_d = 1.0f / (float)a.D;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x);
    const uint8_t* gy = reinterpret_cast<const uint8_t*>(a.gy);
    constexpr int xs = XB ? 2 : 4, gs = GB ? 2 : 4;
    int64_t m = (int64_t)blockIdx.x * TEAMS + mine;
    Raw<XB> cx[NV];
    Raw<GB> cg[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto request = [&](int64_t row) {
        const int end = row < a.M ? a.D : 0;  // (a team without a row left takes part in the barriers with zeros)
        rstd = 0.0f;
        if (row < a.M) mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            fetch<XB, VEC>(cx[v], x + row * a.D * xs, first_index<T, VEC>(t, v), end);
            fetch<GB, VEC>(cg[v], gy + row * a.D * gs, first_index<T, VEC>(t, v), end);
        }
    };
    if constexpr (AHEAD) request(m);
    float w[NV][8], dg[NV][8], db[NV][8];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        Raw<false> r;
#pragma unroll
        for (int i = 0; i < 8; i++) w[v][i] = 1.0f, dg[v][i] = 0.0f, db[v][i] = 0.0f;
        if (a.gamma) fetch<false, VEC>(r, a.gamma, first_index<T, VEC>(t, v), a.D), widen<false>(r, w[v]);
    }
    for (int32_t k = 0; k < rounds; k++, m += teams) {
        float xh[NV][8], f[NV][8];
        if constexpr (!AHEAD) request(m);
        const float rs = rstd;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            widen<XB>(cx[v], xh[v]);
            widen<GB>(cg[v], f[v]);
            const int at = first_index<T, VEC>(t, v);
            const float rv = !VEC || at < a.D ? rs : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // (behind the row, and for a team without one, gy is zero and rstd counts as zero: a mean beyond
                // 2^128 / rstd times that zero would be a NaN in every sum)
                xh[v][i] = VEC || at + 16 * i < a.D ? (xh[v][i] - mean) * rv : 0.0f;
                dg[v][i] += f[v][i] * xh[v][i];
                db[v][i] += f[v][i];
                f[v][i] *= w[v][i];
                s1 += f[v][i];
                s2 += f[v][i] * xh[v][i];
            }
        }
        const int64_t row = m;
        if constexpr (AHEAD)
            if (k + 1 < rounds) request(m + teams);
        float c1 = wave_sum(s1), c2 = wave_sum(s2);
        if constexpr (T > 64) {
            float(&at)[2][T / 64] = lds[k & 1][mine];
            if ((threadIdx.x & 63) == 0) at[0][wave] = c1, at[1][wave] = c2;
            __syncthreads();
            c1 = at[0][0], c2 = at[1][0];
#pragma unroll
            for (int q = 1; q < T / 64; q++) c1 += at[0][q], c2 += at[1][q];
        }
        c1 *= inv_d, c2 *= inv_d;
        if (row < a.M) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
#pragma unroll
                for (int i = 0; i < 8; i++) f[v][i] = rs * (f[v][i] - c1 - xh[v][i] * c2);
                put<VEC>(a.gx, a.gx_dtype, row * a.D, first_index<T, VEC>(t, v), a.D, f[v]);
            }
        }
    }
    if (!a.dgamma) return;
    if constexpr (TEAMS > 1) {
        // the last team first, team 0 last: a fixed order, and team 0's own sums stay in registers
        for (int q = TEAMS - 1; q >= 0; q--) {
            if (mine == q) {
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int at = (v * 8 + i) * T + t;
                        if (q < TEAMS - 1) dg[v][i] += meet[at], db[v][i] += meet[W + at];
                        if (q > 0) meet[at] = dg[v][i], meet[W + at] = db[v][i];
                    }
            }
            __syncthreads();
        }
    }
    if (mine == 0) {
        float* out = a.partial + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int k = first_index<T, VEC>(t, v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = VEC ? k + i : k + 16 * i;
                if (d < a.D) out[d] = dg[v][i], out[a.D + d] = db[v][i];
            }
        }
    }
}

// Backward in one launch: workgroups of two kinds, which need nothing of each other, since the statistics are given.  The first
// `columns` take 16 columns each, one value per thread and row, their rows dealt over THREADS / 16 slices whose sums meet in
// LDS in order: dgamma and dbeta, no partials.  The others are teams of T threads, a row each: gx.  x and gy are read twice,
// the second time from L2.
template <int T, int NV, int THREADS, bool XB, bool GB, bool VEC>
__global__ __launch_bounds__(THREADS) void layer_norm_grad_once_kernel(const NormGradArgs a, int32_t columns, int32_t rounds) {
    constexpr int PER = THREADS / T, SLICES = THREADS / 16;
    __shared__ float lds[2][PER][2][T / 64];
    __shared__ float meet[2][SLICES][16];
    if ((int)blockIdx.x < columns) {
        const int c = threadIdx.x % 16, s = threadIdx.x / 16;
        const int64_t d = (int64_t)blockIdx.x * 16 + c;
        float g = 0.0f, b = 0.0f;
        if (d < a.D) {
#pragma unroll 8
            for (int64_t m = s; m < a.M; m += SLICES) {
                const float t = load1(a.gy, GB ? NQ_DT_BF16 : NQ_DT_F32, m * a.D + d);
                g += t * ((load1(a.x, XB ? NQ_DT_BF16 : NQ_DT_F32, m * a.D + d) - a.mean[m]) * a.rstd[m]);
                b += t;
            }
        }
        meet[0][s][c] = g, meet[1][s][c] = b;
        __syncthreads();
        if (s < 2 && d < a.D) {
            float v = 0.0f;
#pragma unroll 8
            for (int q = 0; q < SLICES; q++) v += meet[s][q][c];
            (s == 0 ? a.dgamma : a.dbeta)[d] = v;
        }
        return;
    }
    const int t = threadIdx.x % T, mine = (int)threadIdx.x / T, wave = t / 64;
    const int64_t teams = (int64_t)((int)gridDim.x - columns) * PER;
    const float inv_d = 1.0f / (float)a.D;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x);
    const uint8_t* gy = reinterpret_cast<const uint8_t*>(a.gy);
    constexpr int xs = XB ? 2 : 4, gs = GB ? 2 : 4;
    float w[NV][8];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        Raw<false> r;
#pragma unroll
        for (int i = 0; i < 8; i++) w[v][i] = 1.0f;
        if (a.gamma) fetch<false, VEC>(r, a.gamma, first_index<T, VEC>(t, v), a.D), widen<false>(r, w[v]);
    }
    int64_t m = (int64_t)((int)blockIdx.x - columns) * PER + mine;
    for (int32_t k = 0; k < rounds; k++, m += teams) {
        const int end = m < a.M ? a.D : 0;  // (a team without a row left takes part in the barriers with zeros)
        Raw<XB> rx[NV];
        Raw<GB> rg[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            fetch<XB, VEC>(rx[v], x + m * a.D * xs, first_index<T, VEC>(t, v), end);
            fetch<GB, VEC>(rg[v], gy + m * a.D * gs, first_index<T, VEC>(t, v), end);
        }
        const float mean = end > 0 ? a.mean[m] : 0.0f, rstd = end > 0 ? a.rstd[m] : 0.0f;
        float xh[NV][8], f[NV][8];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            widen<XB>(rx[v], xh[v]);
            widen<GB>(rg[v], f[v]);
            const int at = first_index<T, VEC>(t, v);
            const float rv = !VEC || at < a.D ? rstd : 0.0f;  // (behind the row: as in the kernel above)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                xh[v][i] = VEC || at + 16 * i < a.D ? (xh[v][i] - mean) * rv : 0.0f;
                f[v][i] *= w[v][i];
                s1 += f[v][i];
                s2 += f[v][i] * xh[v][i];
            }
        }
        float c1 = wave_sum(s1), c2 = wave_sum(s2);
        if constexpr (T > 64) {
            float(&at)[2][T / 64] = lds[k & 1][mine];
            if ((threadIdx.x & 63) == 0) at[0][wave] = c1, at[1][wave] = c2;
            __syncthreads();
            c1 = at[0][0], c2 = at[1][0];
#pragma unroll
            for (int q = 1; q < T / 64; q++) c1 += at[0][q], c2 += at[1][q];
        }
        c1 *= inv_d, c2 *= inv_d;
#pragma unroll
        for (int v = 0; v < NV; v++) {
#pragma unroll
            for (int i = 0; i < 8; i++) f[v][i] = rstd * (f[v][i] - c1 - xh[v][i] * c2);
            put<VEC>(a.gx, a.gx_dtype, m * a.D, first_index<T, VEC>(t, v), end, f[v]);
        }
    }
}

// rows beyond 16384 values: gx, one workgroup per row, two passes
__global__ __launch_bounds__(1024) void layer_norm_grad_x_long_kernel(const NormGradArgs a) {
    __shared__ float lds[2][16];
    const int wave = threadIdx.x / 64;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const int64_t base = m * a.D;
        const float mean = a.mean[m], rstd = a.rstd[m];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t d = threadIdx.x; d < a.D; d += 1024) {
            const float t = load1(a.gy, a.gy_dtype, base + d) * (a.gamma ? a.gamma[d] : 1.0f);
            s1 += t;
            s2 += t * ((load1(a.x, a.x_dtype, base + d) - mean) * rstd);
        }
        const float c1 = team_sum<1024>(s1, lds[0], wave) / (float)a.D, c2 = team_sum<1024>(s2, lds[1], wave) / (float)a.D;
        for (int64_t d = threadIdx.x; d < a.D; d += 1024) {
            const float t = load1(a.gy, a.gy_dtype, base + d) * (a.gamma ? a.gamma[d] : 1.0f);
            const float xh = (load1(a.x, a.x_dtype, base + d) - mean) * rstd;
            store1(a.gx, a.gx_dtype, base + d, rstd * (t - c1 - xh * c2));
        }
    }
}
// ... and the partials: one thread per column and slice of rows
__global__ __launch_bounds__(64) void layer_norm_grad_w_long_kernel(const NormGradArgs a) {
    const int64_t d = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (d >= a.D) return;
    float g = 0.0f, b = 0.0f;
    for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y) {
        const float t = load1(a.gy, a.gy_dtype, m * a.D + d);
        g += t * ((load1(a.x, a.x_dtype, m * a.D + d) - a.mean[m]) * a.rstd[m]);
        b += t;
    }
    a.partial[(int64_t)blockIdx.y * 2 * a.D + d] = g;
    a.partial[(int64_t)blockIdx.y * 2 * a.D + a.D + d] = b;
}

// dgamma | dbeta = the sum of P partials [2 D]: 64 columns x 16 slices of P per workgroup, the slices added in order
__global__ __launch_bounds__(1024) void layer_norm_grad_sum_kernel(const float* __restrict__ partial, float* __restrict__ dgamma,
                                                                   float* __restrict__ dbeta, int32_t D, int32_t P) {
    __shared__ float part[16][64];
    const int c = threadIdx.x & 63, s = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + c, n = 2 * (int64_t)D;
    float v = 0.0f;
    if (col < n) {
        const float* p = partial + col;
#pragma unroll 4
        for (int k = s; k < P; k += 16) v += p[k * n];
    }
    part[s][c] = v;
    __syncthreads();
    if (s == 0 && col < n) {
#pragma unroll
        for (int k = 1; k < 16; k++) v += part[k][c];
        if (col < D)
            dgamma[col] = v;
        else
            dbeta[col - D] = v;
    }
}

__global__ __launch_bounds__(256) void zero_kernel(float* p, float* q, int32_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0.0f, q[i] = 0.0f;
}

constexpr int MAX_HELD = 16384;

// threads per row and vectors per thread: backward with partials
void grad_team_of(int32_t D, int* T, int* NV) {
    *T = D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024;
    *NV = D <= *T * 8 ? 1 : 2;
}

// ... and forward
void team_of(int32_t D, int* T, int* NV) {
    *T = D <= 1024 ? 64 : D <= 4096 ? 256 : D <= 8192 ? 512 : 1024;
    *NV = D <= *T * 8 ? 1 : 2;
}

template <int T, int NV>
int32_t launch_norm(const NormArgs& a, hipStream_t s) {
    // As many workgroups as the chip holds at once (2048 threads per CU); a team then walks M / teams rows
    constexpr int THREADS = T < 256 ? 256 : T, PER = THREADS / T;
    const int64_t want = ((int64_t)a.M + PER - 1) / PER;
    const int32_t grid = (int32_t)std::min<int64_t>(want, 256 * (2048 / THREADS));
    const bool bf16 = a.x_dtype == NQ_DT_BF16, vec = a.D % 8 == 0;
#define NQ_LN(B, V) hipLaunchKernelGGL((layer_norm_kernel<T, NV, B, V>), dim3(grid), dim3(THREADS), 0, s, a, grid * PER)
    if (bf16 && vec) NQ_LN(true, true);
    else if (bf16) NQ_LN(true, false);
    else if (vec) NQ_LN(false, true);
    else NQ_LN(false, false);
#undef NQ_LN
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

// Where both gradients come from one launch and no partials (layer_norm_grad_once_kernel): its columns take a time that grows
// with M / slices, and the rows are read twice.  Partials / one launch, us, in fp32 (bf16 in brackets): 1 x 960 7.4 / 4.4 (a
// launch saved), 333 x 1001 9.0 / 4.4 (8.9 / 3.5), 1024 x 960 9.9 / 7.3 (8.6 / 6.8), 2048 x 960 13.2 / 12.6 (10.4 / 10.9), 512 x 4096
// 18.4 / 10.0 (16.1 / 8.7), 1024 x 4096 20.6 / 18.3 (17.8 / 14.8), 1536 x 4096 25.7 / 27.4 (17.5 / 21.8), 1024 x 8192 47.8 / 36.7
// (37.4 / 29.5), 1024 x 11008 51.9 / 54.4 (37.0 / 38.2); rows of odd length, whose columns lie across lines: 512 x 4095 15.6 / 12.0
// (14.5 / 10.2), 1024 x 4095 18.5 / 23.2 (17.4 / 18.7), 333 x 8191 17.1 / 18.2 (18.5 / 17.8), but 512 x 11007 39.4 / 36.2 (37.1 /
// 29.9; the other kernel's 16 values per thread need 84 bytes of scratch memory there).
bool grad_once(int32_t M, int32_t D) {
    return D <= MAX_HELD && M <= 1024 && (int64_t)M * D <= (D % 8 == 0 || D > 8192 ? 1 << 23 : 1 << 21);
}

// workgroups of the other kernels, one per CU, fewer where the rows run out: as many partials
int32_t grad_workgroups(int32_t M, int32_t D) {
    if (D > MAX_HELD) return (int32_t)std::min<int64_t>(64, ((int64_t)M + 63) / 64);
    int T, NV;
    grad_team_of(D, &T, &NV);
    const int64_t teams = 1024 / T;
    return (int32_t)std::min<int64_t>(256, (M + teams - 1) / teams);
}

template <int T, int NV, bool XB, bool GB>
int32_t launch_grad_types(const NormGradArgs& a, int32_t P, hipStream_t s) {
    constexpr int TEAMS = 1024 / T;
    static LdsAttrOnce attr[2];
    const size_t lds = TEAMS > 1 && a.dgamma ? (size_t)2 * T * 8 * NV * 4 : 0;
    const int32_t rounds = (int32_t)(((int64_t)a.M + (int64_t)P * TEAMS - 1) / ((int64_t)P * TEAMS));
    if (a.D % 8 == 0) {
        NQ_HIP(set_max_lds_once(attr[0], reinterpret_cast<const void*>(&layer_norm_grad_kernel<T, NV, XB, GB, true>), (size_t)2 * T * 8 * NV * 4));
        hipLaunchKernelGGL((layer_norm_grad_kernel<T, NV, XB, GB, true>), dim3(P), dim3(1024), lds, s, a, rounds);
    } else {
        NQ_HIP(set_max_lds_once(attr[1], reinterpret_cast<const void*>(&layer_norm_grad_kernel<T, NV, XB, GB, false>), (size_t)2 * T * 8 * NV * 4));
        hipLaunchKernelGGL((layer_norm_grad_kernel<T, NV, XB, GB, false>), dim3(P), dim3(1024), lds, s, a, rounds);
    }
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

template <int T, int NV>
int32_t launch_grad(const NormGradArgs& a, int32_t P, hipStream_t s) {
    const bool xb = a.x_dtype == NQ_DT_BF16, gb = a.gy_dtype == NQ_DT_BF16;
    if (xb && gb) return launch_grad_types<T, NV, true, true>(a, P, s);
    if (xb) return launch_grad_types<T, NV, true, false>(a, P, s);
    if (gb) return launch_grad_types<T, NV, false, true>(a, P, s);
    return launch_grad_types<T, NV, false, false>(a, P, s);
}

int32_t launch_grad_held(const NormGradArgs& a, int32_t P, hipStream_t s) {
    int T, NV;
    grad_team_of(a.D, &T, &NV);
    switch (T) {
        case 64: return launch_grad<64, 1>(a, P, s);
        case 128: return launch_grad<128, 1>(a, P, s);
        case 256: return launch_grad<256, 1>(a, P, s);
        case 512: return launch_grad<512, 1>(a, P, s);
        default: return NV == 1 ? launch_grad<1024, 1>(a, P, s) : launch_grad<1024, 2>(a, P, s);
    }
}

template <int T, int NV, int THREADS>
int32_t launch_once(const NormGradArgs& a, bool columns, bool rows, hipStream_t s) {
    constexpr int64_t PER = THREADS / T;
    const int32_t nc = columns ? (a.D - 1) / 16 + 1 : 0;
    const int32_t nr = rows ? (int32_t)std::min<int64_t>((a.M + PER - 1) / PER, 256 * (2048 / THREADS)) : 0;
    const int32_t rounds = rows ? (int32_t)((a.M + nr * PER - 1) / (nr * PER)) : 0;
    const bool xb = a.x_dtype == NQ_DT_BF16, gb = a.gy_dtype == NQ_DT_BF16, vec = a.D % 8 == 0;
#define NQ_GO(X, G, V) \
    hipLaunchKernelGGL((layer_norm_grad_once_kernel<T, NV, THREADS, X, G, V>), dim3(nc + nr), dim3(THREADS), 0, s, a, nc, rounds)
#define NQ_GV(X, G)             \
    if (vec) NQ_GO(X, G, true); \
    else NQ_GO(X, G, false)
    if (xb && gb) { NQ_GV(true, true); }
    else if (xb) { NQ_GV(true, false); }
    else if (gb) { NQ_GV(false, true); }
    else { NQ_GV(false, false); }
#undef NQ_GV
#undef NQ_GO
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

int32_t launch_grad_once(const NormGradArgs& a, bool columns, bool rows, hipStream_t s) {
    if (a.D <= 512) return launch_once<64, 1, 1024>(a, columns, rows, s);
    if (a.D <= 2048) return launch_once<256, 1, 512>(a, columns, rows, s);
    if (a.D <= 4096) return launch_once<512, 1, 512>(a, columns, rows, s);
    if (a.D <= 8192) return launch_once<1024, 1, 1024>(a, columns, rows, s);
    return launch_once<1024, 2, 1024>(a, columns, rows, s);
}

}  // namespace

int32_t launch_layer_norm(const NormArgs& a, hipStream_t s) {
    if (a.D > MAX_HELD) {
        hipLaunchKernelGGL(layer_norm_long_kernel, dim3((unsigned)std::min(a.M, 1 << 20)), dim3(1024), 0, s, a);
        NQ_HIP(hipGetLastError());
        return NQ_OK;
    }
    int T, NV;
    team_of(a.D, &T, &NV);
    switch (T * 4 + NV) {
        case 64 * 4 + 1: return launch_norm<64, 1>(a, s);
        case 64 * 4 + 2: return launch_norm<64, 2>(a, s);
        case 256 * 4 + 1: return launch_norm<256, 1>(a, s);
        case 256 * 4 + 2: return launch_norm<256, 2>(a, s);
        case 512 * 4 + 2: return launch_norm<512, 2>(a, s);
        default: return launch_norm<1024, 2>(a, s);
    }
}

int64_t layer_norm_grad_partial_bytes(int32_t M, int32_t D) { return grad_once(M, D) ? 0 : (int64_t)grad_workgroups(M, D) * 2 * D * 4; }

int32_t launch_layer_norm_grad(const NormGradArgs& a, hipStream_t s) {
    if (a.M == 0) {
        if (!a.dgamma) return NQ_OK;
        hipLaunchKernelGGL(zero_kernel, dim3((unsigned)((a.D - 1) / 256 + 1)), dim3(256), 0, s, a.dgamma, a.dbeta, a.D);
        NQ_HIP(hipGetLastError());
        return NQ_OK;
    }
    if (grad_once(a.M, a.D)) {
        // (gx written over what the columns read: they go first, in a launch of their own; gx has the same bits either way)
        const bool over = a.gx == a.x || a.gx == a.gy;
        if (a.dgamma && over) {
            const int32_t rc = launch_grad_once(a, true, false, s);
            if (rc) return rc;
        }
        return launch_grad_once(a, a.dgamma && !over, true, s);
    }
    const int32_t P = grad_workgroups(a.M, a.D);
    if (a.D > MAX_HELD) {
        if (a.dgamma) {  // (the columns first: gx may be gy's own memory)
            hipLaunchKernelGGL(layer_norm_grad_w_long_kernel, dim3((unsigned)((a.D - 1) / 64 + 1), (unsigned)P), dim3(64), 0, s, a);
            NQ_HIP(hipGetLastError());
        }
        hipLaunchKernelGGL(layer_norm_grad_x_long_kernel, dim3((unsigned)std::min(a.M, 1 << 20)), dim3(1024), 0, s, a);
        NQ_HIP(hipGetLastError());
    } else {
        const int32_t rc = launch_grad_held(a, P, s);
        if (rc) return rc;
    }
    if (a.dgamma) {
        hipLaunchKernelGGL(layer_norm_grad_sum_kernel, dim3((unsigned)((2 * (int64_t)a.D - 1) / 64 + 1)), dim3(1024), 0, s, a.partial, a.dgamma,
                           a.dbeta, a.D, P);
        NQ_HIP(hipGetLastError());
    }
    return NQ_OK;
}

}  // namespace nq
