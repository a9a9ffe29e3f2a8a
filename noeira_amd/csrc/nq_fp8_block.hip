// The block-scaled fp8 linear (NQ_FMT_FP8_BLOCK):
//     y[m, n] = epi( sum_g sx[m, g] sw[n / 128, g] * sum_{k in block g} qx[m, k] qw[n, k]  + bias[n] )
// with e4m3 codes qx, qw, one fp32 scale per activation row and 128 of K and one per 128 x 128 block of the weight.
//
// Why the block is the unit of everything here.  One v_mfma_f32_16x16x128_f8f6f4 multiplies 16 weight rows by 16
// activation rows over exactly 128 k: its result is one block's sum for 256 outputs, summed by the matrix core from a
// zero addend, and the two scales enter as ONE fused multiply-add per output and block.  With the weight as the
// first operand a lane holds one activation row and four consecutive channels, so the row's scale is a lane's own
// value, the weight's is the same for all lanes, and their product is made once per lane and block.
//
// Which matrix core.  The fp8 one does not sum in full fp32.  On this GPU it adds the products of eight adjacent k under
// one exponent, the largest sum e of two codes' exponents among them (-6 for subnormal codes), and cuts each product to a
// multiple of 2^(e - 13), towards zero; the groups' sums are then added in fp32.  (A single product beside a cancelling
// pair of 256 * 256 in its group: 8 comes out as 8, 15 as 8, 7.5 as 0; in another group down to 2^-7.)  So a block's sum is off
// by 7 * 2^-13 = 8.5e-4 of the sum of the products' magnitudes at worst (rows and weights made for it reach 8.4e-4; a
// subnormal code has up to 2^3 less than its exponent says, two of them 2^6), by 2.2e-4 at most over two million blocks of
// uniformly drawn codes, and by 1.3e-5 of the sums' root mean square for codes of N(0, 1) values (all fp8 shapes alike;
// 5e-5 for uniform codes), where the bf16 one is off by 1e-8.  That is far below what rounding a value to e4m3 costs each term
// (2^-4), and below a bf16 output's half step (2^-8) unless the terms cancel: 8192 x 4096 -> 11008 is off by 1.65890e-3
// of the result's norm where fp32 sums give 1.65888e-3, with 1.3 % of the outputs one step of bf16 apart.  In an fp32 output
// it would be the whole error.  So a call with an fp32 y decodes both operands' codes to bf16, which is exact, and
// multiplies on v_mfma_f32_16x16x32_bf16 (half the rate, and 16 conversions per operand of 16 rows), and a call with a bf16 y
// multiplies the codes.
//
// Weight layout.  The codes are kept only in the matrix core's operand order: tile (R, g) = rows 16 R .., k = 128 g ..
// is 2 KiB at ((R * G) + g) * 2 KiB; lane l = r + 16 c of its first KiB holds row r's k = 16 c .. 16 c + 15, of its
// second k = 64 + 16 c .. 64 + 16 c + 15, both 16 bytes at 16 l.  A wavefront's 128-bit load is one contiguous KiB and
// needs no exchange between lanes.  (Which of the 128 k a lane multiplies is free as long as both operands agree; with
// these a lane's loads of the row-ordered activations are 64 adjacent bytes per row and instruction.)  Rows behind
// OUT and k behind IN are zero.
#include "nq_fp8_block.h"
#include "nq_fp8_quant.h"

#include <algorithm>

namespace nq {

namespace {

// ---- load time ----------------------------------------------------------------------------------------------------

// row-ordered codes [rows][cols] -> tiles; TRANSPOSE: of the transposed matrix (tile rows run along cols).  One thread
// per 16 bytes of a tile.
template <bool TRANSPOSE>
__global__ __launch_bounds__(256) void fp8_block_repack_kernel(const uint8_t* __restrict__ codes, uint8_t* __restrict__ tiles,
                                                               int32_t rows, int32_t cols, int64_t pieces) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= pieces) return;
    const int32_t trows = TRANSPOSE ? cols : rows, tcols = TRANSPOSE ? rows : cols;
    const int32_t G = (tcols - 1) / 128 + 1;
    const int lane = (int)(t & 63), half = (int)(t >> 6) & 1;
    const int64_t tile = t >> 7;
    const int64_t row = tile / G * 16 + (lane & 15);
    const int64_t k0 = tile % G * 128 + 64 * half + 16 * (lane >> 4);
    uint32_t w[4] = {0, 0, 0, 0};
    if (row < trows) {
#pragma unroll
        for (int b = 0; b < 16; b++) {
            const int64_t k = k0 + b;
            if (k < tcols) w[b / 4] |= (uint32_t)codes[TRANSPOSE ? k * cols + row : row * cols + k] << (8 * (b % 4));
        }
    }
    reinterpret_cast<uint4*>(tiles)[t] = make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ __launch_bounds__(256) void fp8_block_scales_t_kernel(const float* __restrict__ s, float* __restrict__ st, int32_t nb,
                                                                 int32_t kb) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t < (int64_t)nb * kb) st[t % kb * nb + t / kb] = s[t];
}

// one thread per 16 values of a row
__global__ __launch_bounds__(256) void fp8_block_dequantize_kernel(const uint8_t* __restrict__ tiles, const float* __restrict__ ws,
                                                                   float* __restrict__ out, int32_t N, int32_t K, int32_t G) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int32_t pieces = K / 16;
    if (t >= (int64_t)N * pieces) return;
    const int64_t n = t / pieces;
    const int32_t k = (int32_t)(t % pieces) * 16, g = k / 128, c = k / 16 % 4, half = k / 64 % 2;
    const uint4 v = *reinterpret_cast<const uint4*>(tiles + (n / 16 * G + g) * 2048 + half * 1024 + (n % 16 + 16 * c) * 16);
    const float s = ws[n / 128 * G + g];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float4* o = reinterpret_cast<float4*>(out + n * K + k);
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = make_float4(__builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * s, __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * s,
                           __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * s, __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * s);
}

// ---- activations --------------------------------------------------------------------------------------------------

// One read and one write of everything: 8192 x 4096 in bf16, 102 MB, 17.6 us = 5.8 TB/s.
// 16 lanes per block of 128.  VEC (K % 8 == 0): a lane's 8 values are adjacent, 128-bit loads and one 64-bit store;
// otherwise every 16th value, element by element.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_fp8_block_kernel(const void* __restrict__ x, uint8_t* __restrict__ codes,
                                                                      float* __restrict__ scales, int32_t K, uint32_t G,
                                                                      uint32_t blocks) {
    const int l = threadIdx.x & 15;
    // (16 lanes, a DPP row, enter and leave together; more than one turn only beyond 2^24 workgroups)
    for (uint32_t b = blockIdx.x * 16u + (threadIdx.x >> 4); b < blocks; b += gridDim.x * 16u) {
        const uint32_t m = b / G, g = b - m * G;
        const int64_t base = (int64_t)m * K;
        float v[8];
        float s;
        if constexpr (VEC) {
            const int32_t k = (int32_t)g * 128 + 8 * l;
            const bool in = k < K;
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.0f;
            if (in) {
                if constexpr (BF16) {
                    const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + base + k);
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
                } else {
                    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + base + k);
                    const float4 a = p[0], c = p[1];
                    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = c.x, v[5] = c.y, v[6] = c.z, v[7] = c.w;
                }
            }
            const uint2 q = quantize_block16(v, s);
            if (in) *reinterpret_cast<uint2*>(codes + base + k) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int32_t k = (int32_t)g * 128 + 16 * i + l;
                const int64_t at = base + min(k, K - 1);  // (no branch per load, behind which each would be waited for)
                const float w = BF16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(x)[at] << 16)
                                     : reinterpret_cast<const float*>(x)[at];
                v[i] = k < K ? w : 0.0f;
            }
            const uint2 q = quantize_block16(v, s);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int32_t k = (int32_t)g * 128 + 16 * i + l;
                if (k < K) codes[base + k] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
            }
        }
        if (l == 0) scales[b] = s;
    }
}

// ---- the product --------------------------------------------------------------------------------------------------

// Few rows: MT x NT MFMA tiles of 16 x 16 per workgroup, the blocks of K dealt over KW wavefronts, whose sums meet in LDS
// in wavefront order (bit-repeatable).  U: blocks requested together.  Both operands go from memory to registers: the
// weight's tiles are contiguous, every byte of them is read once per 16 MT rows, and at one row nothing else matters.
// One row over 4096 -> 11008 (45 MB, rotating over copies): 9.1 us in bf16, 4.9 TB/s (a plain copy moves 5.0); 256 rows over
// 4096 -> 4096: 15.2, 134 MB from L2 at 11 TB/s.  That is the rate of these loads, 64 bytes of a row of x at a time, and it
// bounds the calls from about 16 rows on; it is not the path's: transfers into LDS reach 16 - 21 TB/s in the GEMMs of this
// library.  (64 / 128 / 256 rows: 2.4 / 3.4 / 3.9 times the floor of their bytes and products.)
template <int MT, int NT, int KW, int U, bool EXACT>
__global__ __launch_bounds__(64 * KW) void fp8_block_tile_kernel(const BlockParams p) {
    constexpr int ROWS = 16 * MT, CH = 16 * NT;
    extern __shared__ __attribute__((aligned(16))) uint8_t meet[];
    float(*const part)[ROWS][CH + 4] = reinterpret_cast<float(*)[ROWS][CH + 4]>(meet);  // [KW]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int tn = blockIdx.x / p.tiles_m, tm = blockIdx.x - tn * p.tiles_m;
    const int m0 = tm * ROWS, n0 = tn * CH;
    const int row_tiles = (p.N + 15) / 16;

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // rows behind M repeat the last one: their results are columns of their own, never stored
    int64_t mrow[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) mrow[i] = min(m0 + 16 * i + r, p.M - 1);
    const uint8_t* wtile[NT];
    const float* wscale[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int R = min(n0 / 16 + j, row_tiles - 1);
        wtile[j] = p.w + (int64_t)R * p.G * 2048 + lane * 16;
        wscale[j] = p.ws + (int64_t)(R / 8) * p.G;
    }
    static_assert(4 % U == 0, "scales come four blocks at a time");
    for (int four = wave; four < p.G; four += 4 * KW) {
        // a row's scales of the next four blocks, one per lane that holds the row: one request for 16 rows instead of four
        // (16 lines each; as requests of every block's own they were a fifth of those under way)
        float sx4[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) sx4[i] = p.xs[mrow[i] * p.G + min(four + c * KW, p.G - 1)];
#pragma unroll
        for (int b = 0; b < 4; b += U) {
            const int g0 = four + b * KW;
            if (g0 >= p.G) break;
            i32x4 xv[U][MT][2], wv[U][NT][2];
            float sw[U][NT];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int g = min(g0 + u * KW, p.G - 1);
#pragma unroll
                for (int j = 0; j < NT; j++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) wv[u][j][e] = *reinterpret_cast<const i32x4*>(wtile[j] + (int64_t)g * 2048 + e * 1024);
                    sw[u][j] = wscale[j][g];
                }
#pragma unroll
                for (int i = 0; i < MT; i++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        // (K is a multiple of 16: a piece lies in the row or behind it, and what lies behind counts as zero)
                        const int k = 128 * g + 64 * e + 16 * c;
                        const i32x4 v = *reinterpret_cast<const i32x4*>(p.x + mrow[i] * p.K + (k < p.K ? k : 0));
                        xv[u][i][e] = k < p.K ? v : i32x4{0, 0, 0, 0};
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float sx[MT];
#pragma unroll
                for (int i = 0; i < MT; i++)
                    sx[i] = __int_as_float(__builtin_amdgcn_ds_bpermute((r + 16 * (b + u)) * 4, __float_as_int(sx4[i])));
                if (g0 + u * KW < p.G) {
                    Operand<EXACT> w[NT];
#pragma unroll
                    for (int j = 0; j < NT; j++) w[j] = Operand<EXACT>(wv[u][j][0], wv[u][j][1]);
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        const Operand<EXACT> x(xv[u][i][0], xv[u][i][1]);
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            const f32x4 d = block_sum(w[j], x);
                            const float s = sx[i] * sw[u][j];
#pragma unroll
                            for (int t = 0; t < 4; t++) acc[i][j][t] = fmaf(d[t], s, acc[i][j][t]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) *reinterpret_cast<f32x4*>(&part[wave][16 * i + r][16 * j + 4 * c]) = acc[i][j];
    __syncthreads();
    auto finish = [&](float z, int n) {
        if (p.bias)
            z += p.bias_dtype == NQ_DT_F32 ? reinterpret_cast<const float*>(p.bias)[n]
                                           : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p.bias)[n] << 16);
        return p.relu ? (z > 0.0f ? z : 0.0f) : z;
    };
    typedef typename std::conditional<EXACT, float, __bf16>::type out_t;
    void* y;
    int width, col;
    if (p.vec) {  // four channels of a row per thread (OUT % 4 == 0: a part's boundary or end never among them)
        for (int o = threadIdx.x; o < ROWS * CH / 4; o += 64 * KW) {
            const int row = o / (CH / 4), ch = o % (CH / 4) * 4;
            const int m = m0 + row, n = n0 + ch;
            if (m >= p.M || n >= p.N) continue;
            f32x4 z = *reinterpret_cast<const f32x4*>(&part[0][row][ch]);
#pragma unroll
            for (int w = 1; w < KW; w++) z += *reinterpret_cast<const f32x4*>(&part[w][row][ch]);
#pragma unroll
            for (int t = 0; t < 4; t++) z[t] = finish(z[t], n + t);
            seg_lookup(p.seg, n, y, width, col);
            out_t* q = reinterpret_cast<out_t*>(y) + (int64_t)m * width + col;
            if constexpr (EXACT)
                *reinterpret_cast<f32x4*>(q) = z;
            else
                *reinterpret_cast<bf16x4*>(q) = __builtin_convertvector(z, bf16x4);
        }
    } else {  // one channel per thread, adjacent threads adjacent
        for (int o = threadIdx.x; o < ROWS * CH; o += 64 * KW) {
            const int row = o / CH, ch = o % CH;
            const int m = m0 + row, n = n0 + ch;
            if (m >= p.M || n >= p.N) continue;
            float z = part[0][row][ch];
#pragma unroll
            for (int w = 1; w < KW; w++) z += part[w][row][ch];
            seg_lookup(p.seg, n, y, width, col);
            reinterpret_cast<out_t*>(y)[(int64_t)m * width + col] = (out_t)finish(z, n);
        }
    }
}

template <int MT, int NT, int KW, int U>
int32_t launch_tile(BlockParams p, hipStream_t s) {
    p.tiles_m = (p.M - 1) / (16 * MT) + 1;
    const int64_t grid = (int64_t)p.tiles_m * ((p.N - 1) / (16 * NT) + 1);  // (fits a launch: pick_shape)
    constexpr size_t lds = sizeof(float) * KW * 16 * MT * (16 * NT + 4);
    static LdsAttrOnce attr[2];
    if (p.y_dtype == NQ_DT_F32) {
        if (lds > 65536) NQ_HIP(set_max_lds_once(attr[0], reinterpret_cast<const void*>(&fp8_block_tile_kernel<MT, NT, KW, U, true>), lds));
        hipLaunchKernelGGL((fp8_block_tile_kernel<MT, NT, KW, U, true>), dim3((unsigned)grid), dim3(64 * KW), lds, s, p);
    } else {
        if (lds > 65536) NQ_HIP(set_max_lds_once(attr[1], reinterpret_cast<const void*>(&fp8_block_tile_kernel<MT, NT, KW, U, false>), lds));
        hipLaunchKernelGGL((fp8_block_tile_kernel<MT, NT, KW, U, false>), dim3((unsigned)grid), dim3(64 * KW), lds, s, p);
    }
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

// The tile shapes of the few-rows kernel.  A call of it is bound by the operands' way into the CUs: a workgroup brings in
// 16 (MT + NT) rows of K bytes at about 55 KB per microsecond and CU, a workgroup after a CU's first adds its meeting in LDS
// and its stores, and an fp32 y the second half of its products.  Of the shapes the one with the lowest estimate is taken:
// over 200 calls (1 - 2045 rows, K = 96 .. 11008, N = 17 .. 11008, both y) that and the GEMM's estimate together cost 0.9 %
// over the best of all shapes of either kernel in the mean, 21 % at worst.  Measured (K = N = 4096, M = 16 / 64 / 128 / 256 in bf16,
// us): 1 x 1 5.0 / - / - / -, 1 x 2 5.5 / - / - / -, 2 x 2 - / 7.9 / 13.0 / 23, 2 x 4 - / 9.5 / 12.2 / 21, 4 x 4 - / 13.7 / - / 15.2.
struct Shape {
    int mt, nt;
};
constexpr Shape SHAPES[] = {{1, 1}, {1, 2}, {2, 2}, {2, 4}, {4, 4}};
int64_t tile_workgroups(const BlockParams& p, const Shape& t) {
    return (int64_t)((p.M - 1) / (16 * t.mt) + 1) * ((p.N - 1) / (16 * t.nt) + 1);
}
// K over 16 wavefronts where each keeps two blocks and more and few rows are read: such a call is bound by the loads
// under way (1 row, 4096 -> 11008: 9.5 us against 9.9 on 8; 8 rows, 11008 -> 4096: 10.1 against 11.1; 16: 13.6 against 11.8)
int tile_wavefronts(const BlockParams& p, const Shape& t) {
    return t.mt * t.nt == 1 && (p.M == 1 ? p.G >= 32 : p.M <= 8 && p.G >= 64) ? 16 : 8;
}
double tile_estimate_us(const BlockParams& p, const Shape& t) {
    const int64_t wgs = tile_workgroups(p, t);
    const double per_cu = (double)((wgs + 255) / 256), tiles = t.mt * t.nt;
    const double one = (double)p.K * (16.0 * (t.mt + t.nt) / 55e3 + (p.y_dtype == NQ_DT_F32 ? 9e-6 * tiles : 0.0));
    return 2.9 + 0.10 * tiles + per_cu * one + (per_cu - 1.0) * 0.19 * tiles;
}
// ... or null, where none is one launch of fewer than 2^32 threads
const Shape* pick_shape(const BlockParams& p, double* us) {
    const Shape* best = nullptr;
    for (const Shape& t : SHAPES) {
        if (16 * (t.mt - 1) >= p.M) break;  // (no tile of rows that are not there)
        if (tile_workgroups(p, t) * 64 * tile_wavefronts(p, t) > UINT32_MAX) continue;
        const double e = tile_estimate_us(p, t);
        if (!best || e < *us) best = &t, *us = e;
    }
    return best;
}
// the few-rows kernel's shape, or null for the GEMM
int32_t pick_kernel(const BlockParams& p, const Shape** shape) {
    double tile_us = 0.0;
    *shape = pick_shape(p, &tile_us);
    double gemm_us = 0.0;
    if (!fp8_block_gemm_estimate_us(p, &gemm_us)) {
        if (*shape) return NQ_OK;
        return fail(NQ_ERR_INVALID, "FP8_BLOCK product: " + std::to_string(p.M) + " rows of " + std::to_string(p.N) +
                                        " outputs are too many for one launch");
    }
    if (*shape && gemm_us < tile_us) *shape = nullptr;
    return NQ_OK;
}

}  // namespace

int32_t launch_fp8_block_repack(const uint8_t* codes, uint8_t* tiles, int32_t rows, int32_t cols, bool transpose, hipStream_t s) {
    const int64_t trows = transpose ? cols : rows, tcols = transpose ? rows : cols;
    const int64_t pieces = (trows + 15) / 16 * ((tcols + 127) / 128) * 128;
    if (transpose)
        hipLaunchKernelGGL((fp8_block_repack_kernel<true>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, codes, tiles, rows, cols, pieces);
    else
        hipLaunchKernelGGL((fp8_block_repack_kernel<false>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, codes, tiles, rows, cols, pieces);
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

int32_t launch_fp8_block_scales_t(const float* scales, float* scales_t, int32_t nb, int32_t kb, hipStream_t s) {
    const int64_t n = (int64_t)nb * kb;
    hipLaunchKernelGGL(fp8_block_scales_t_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, scales, scales_t, nb, kb);
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

int32_t launch_fp8_block_dequantize(const nq_layer* L, float* out, hipStream_t s) {
    const int64_t n = (int64_t)L->out * (L->in / 16);
    hipLaunchKernelGGL(fp8_block_dequantize_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, L->d_codes,
                       reinterpret_cast<const float*>(L->d_scales), out, L->out, L->in, L->groups);
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

int32_t launch_quantize_rows_fp8_block(const void* x, int32_t x_dtype, uint8_t* codes, float* scales, int32_t M, int32_t K,
                                       hipStream_t s) {
    const int64_t G = (K - 1) / 128 + 1, blocks = M * G;
    if (blocks > INT32_MAX) return fail(NQ_ERR_INVALID, "nq_quantize_rows_fp8_block: more than 2^31 - 1 blocks of 128");
    const bool bf16 = x_dtype == NQ_DT_BF16, vec = K % 8 == 0;
#define NQ_QB(B, V)                                                                                                        \
    hipLaunchKernelGGL((quantize_rows_fp8_block_kernel<B, V>), dim3((unsigned)std::min<int64_t>((blocks + 15) / 16, (1 << 24) - 1)), \
                       dim3(256), 0, s, x, codes, scales, K, (uint32_t)G, (uint32_t)blocks)
    if (bf16 && vec) NQ_QB(true, true);
    else if (bf16) NQ_QB(true, false);
    else if (vec) NQ_QB(false, true);
    else NQ_QB(false, false);
#undef NQ_QB
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

int32_t fp8_block_form(int32_t M, int32_t out, int32_t in, int32_t y_dtype, int32_t* form) {
    BlockParams p{};
    p.M = M, p.N = out, p.K = in, p.G = (in - 1) / FP8_BLOCK + 1, p.y_dtype = y_dtype;
    const Shape* shape = nullptr;
    if (const int32_t rc = pick_kernel(p, &shape)) return rc;
    if (!shape) {
        fp8_block_gemm_form(p, form);
        return NQ_OK;
    }
    form[0] = 0, form[1] = 16 * shape->mt, form[2] = 16 * shape->nt, form[3] = tile_wavefronts(p, *shape), form[4] = 0;
    return NQ_OK;
}

int32_t launch_fp8_block(const ForwardArgs& a) {
    const nq_layer* L = a.L;
    int device = -1;
    NQ_HIP(hipGetDevice(&device));
    if (device != L->device)
        return fail(NQ_ERR_INVALID, "layer was loaded on device " + std::to_string(L->device) + " but the current device is " + std::to_string(device));
    BlockParams p{};
    p.x = reinterpret_cast<const uint8_t*>(a.x), p.w = L->d_codes;
    p.xs = a.x_scale, p.ws = reinterpret_cast<const float*>(L->d_scales), p.bias = a.bias;
    p.M = a.M, p.N = L->out, p.K = L->in, p.G = L->groups;
    p.y_dtype = a.y_dtype, p.bias_dtype = a.bias_dtype, p.relu = a.epilogue == NQ_EPI_RELU;
    p.seg = a.seg;
    const uintptr_t line = a.y_dtype == NQ_DT_F32 ? 15 : 7;  // four channels of y
    p.vec = L->out % 4 == 0;
    for (int t = 0; t < a.seg.nseg; t++) p.vec = p.vec && ((uintptr_t)a.seg.y[t] & line) == 0;
    const Shape* shape = nullptr;
    if (const int32_t rc = pick_kernel(p, &shape)) return rc;
    if (!shape) return launch_fp8_block_gemm(p, a.stream);
    switch (shape->mt * 8 + shape->nt) {
        case 1 * 8 + 1:
            if (tile_wavefronts(p, *shape) == 16) return launch_tile<1, 1, 16, 2>(p, a.stream);
            return launch_tile<1, 1, 8, 2>(p, a.stream);
        case 1 * 8 + 2: return launch_tile<1, 2, 8, 2>(p, a.stream);
        case 2 * 8 + 2: return launch_tile<2, 2, 8, 2>(p, a.stream);
        case 2 * 8 + 4: return launch_tile<2, 4, 8, 1>(p, a.stream);
        default: return launch_tile<4, 4, 8, 1>(p, a.stream);
    }
}

}  // namespace nq
