// The block-scaled fp8 product for many activation rows (layout and scales: nq_fp8_block.hip):
//     y[m, n] = epi( sum_g sx[m, g] sw[n / 128, g] * sum_{k in block g} qx[m, k] qw[n, k]  + bias[n] )
//
// A stage of the K loop is one block of 128 k: x tile BM x 128 B, weight tile BN x 128 B and their scales, filled straight
// from global memory (global_load_lds) into one of NB stage buffers.  A wavefront owns TI x TJ results of 16 x 16, and its
// channels lie in one block of 128, so its weight scale is one number per stage.
//
// Why these tiles.  The scales make every result pass the vector ALU once per block (a product into registers of its own,
// then four multiply-adds per lane), so the accumulators have to be vector registers: 128 of a wavefront's 256 with two
// wavefronts per SIMD, 64 x 128 per wavefront, 256 x 256 per CU.  (One wavefront per SIMD with twice the registers could
// not address twice the accumulators, and left the matrix core waiting on its own multiply-adds: 31 us against 24 for
// 512 rows over 4096 -> 4096 on 128 x 128 tiles.)  Smaller calls take smaller tiles (estimate() below).
//
// What bounds it, 8192 x 4096 x 4096 in bf16: 119 - 126 us = 2.2 - 2.3 PFLOP/s, what this library's GEMM with one scale per
// tensor takes (120 us) - the board's power limit.  Below that limit (128 workgroups; parts taken out one
// at a time): whole 50 us; without the transfers 42, without the multiply-adds 44, without either 38, the products alone
// 33 (their matrix core time).  The transfers cost what they occupy of LDS (64 KiB in, 192 KiB of fragments out per stage:
// 2048 cycles at 128 B, as many as the products), the multiply-adds about half of their 1024 vector cycles per stage and
// SIMD.  On 128 x 128 tiles LDS is the bound outright (128 KiB per 512 cycles of products: 0.47 us a stage; 18.2 - 20.6 us
// a round at K = 4096).  With an fp32 y the two bf16 products per fp8 one and 16 conversions per fragment take
// 239 - 252 us (1.1 - 1.15 PFLOP/s; a library bf16 product of the same size 232).
#include <algorithm>

#include "nq_fp8_block.h"

namespace nq {

namespace {

// KS = 2: two groups of WM x WN wavefronts, each with stage buffers of its own, take the blocks of K in turn, and the second
// one's results are added to the first one's through LDS at the end.
template <int BM, int BN, int WM, int WN, int NB, int KS, bool EXACT>
__device__ __forceinline__ void block_gemm_body(const BlockParams& p) {
    constexpr int WAVES = WM * WN;  // of a group
    constexpr int TI = BM / WM / 16, TJ = BN / WN / 16;
    constexpr int PAIRS = TJ / 2;
    constexpr int XB = BM * 128, WB = BN * 128, STAGE = XB + WB;  // bytes of a stage
    constexpr int DX = BM / 8 / WAVES, DW = BN / 8 / WAVES;       // transfers of 1 KiB per wavefront and stage
    constexpr int SW = BM / 64;                                   // wavefronts that fetch x's scales; the next one fetches w's
    constexpr int CHUNK_BYTES = BM * 16 + 256;                    // scales of four stages: [BM][4], then [BN / 128][4]
    static_assert(TJ % 2 == 0 && PAIRS % 2 == 0 && BN / WN <= 128 && SW < WAVES && BM % (8 * WAVES) == 0 && BN % (16 * WAVES) == 0, "tile");
    static_assert(NB >= 2 && NB <= 4 && (NB > 2 || PAIRS >= 3), "the places of the transfers; three buffers of scales");
    constexpr int GROUP = NB * STAGE + 3 * CHUNK_BYTES;  // LDS of a group
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_all[];
    const int lane = threadIdx.x & 63;
    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = KS == 1 ? 0 : wave_all / WAVES, wave = KS == 1 ? wave_all : wave_all % WAVES;
    uint8_t* const lds = lds_all + group * GROUP;
    typedef __attribute__((address_space(3))) void lptr_t;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t*)lds_all + group * GROUP;
    const int wm = wave / WN, wn = wave % WN;

    // ---- tile: ids are dealt round-robin to the 8 XCDs, so each XCD is given one contiguous run, and runs walk bands of 8
    // row tiles, so that the tiles an XCD works on share their operands in its L2
    const int nb = gridDim.x, bid = blockIdx.x;
    const int xcd = bid % 8, lid = xcd * (nb / 8) + min(xcd, nb % 8) + bid / 8;
    constexpr int GM = 8;
    const int band = lid / (GM * p.tiles_n), in_band = lid - band * GM * p.tiles_n;
    const int band_rows = min(GM, p.tiles_m - band * GM);
    const int m0 = p.m_base + (band * GM + in_band % band_rows) * BM, n0 = p.n_base + in_band / band_rows * BN;

    // ---- transfers.  x: 8 rows of 128 B per instruction, the 16-byte slots of a row permuted on the way (swz) so that the
    // fragment reads below meet no bank twice; w: 1 KiB of operand order as it lies; scales: one float per lane.
    auto swz = [](int row) { return (((row >> 1) & 7) + 6) & 7; };
    const uint8_t* const xbase = p.x + (int64_t)m0 * p.K;
    uint32_t xoff[DX];
    int32_t xk[DX];  // where the lane's 16 bytes lie in a stage
#pragma unroll
    for (int t = 0; t < DX; t++) {
        const int row = (wave * DX + t) * 8 + lane / 8;
        xk[t] = ((lane % 8) ^ swz(row)) * 16;
        xoff[t] = (uint32_t)(min(m0 + row, p.M - 1) - m0) * (uint32_t)p.K + xk[t];
    }
    const int row_tiles = (p.N + 15) / 16;
    const uint8_t* wtile[DW / 2];  // a tile's two halves are two transfers
#pragma unroll
    for (int t = 0; t < DW / 2; t++) wtile[t] = p.w + (int64_t)min(n0 / 16 + wave * (DW / 2) + t, row_tiles - 1) * p.G * 2048;
    const uint32_t woff = lane * 16;
    // Scales come four stages at a time (a row's four are 16 adjacent bytes; one at a time, 64 rows to an instruction,
    // they cost 3 - 6 % of the call), in three buffers taken in turn: with stage s goes a quarter of the chunk after its
    // own, which has landed with it, a stage ahead of its first use at the latest, and whose buffer held the chunk
    // before stage s's: the stage being multiplied is at most NB <= 4 stages behind s.
    const bool sx_wave = wave < SW, scaling = wave <= SW;
    const float* const sbase = sx_wave ? p.xs + (int64_t)m0 * p.G : p.ws + (int64_t)(n0 / 128) * p.G;
    const int srow_end = sx_wave ? p.M - m0 : (p.N + 127) / 128 - n0 / 128;
    const uint32_t scales0 = NB * STAGE;
    int iq = 0, ichunk = 4;               // what the next stage requested brings along: quarter iq of the chunk from stage ichunk on
    uint32_t ibuf = scales0 + CHUNK_BYTES;  // ... and the buffer it goes to
    auto scale_dma = [&](int quarter, int from, uint32_t buffer) {
        const int row = sx_wave ? (quarter * SW + wave) * 16 + lane / 4 : lane / 4;
        const uint32_t o = ((uint32_t)min(row, srow_end - 1) * (uint32_t)p.G + (uint32_t)min((from + lane % 4) * KS + group, p.G - 1)) * 4;
        const uint32_t m0v = lds0 + buffer + (sx_wave ? (uint32_t)(quarter * SW + wave) * 256 : BM * 16);
        const float* s = sbase;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(m0v), "v"(o), "s"(s) : "memory");
    };
    auto next_scales = [&]() {
        if (scaling) scale_dma(iq, ichunk, ibuf);
        if (++iq == 4) iq = 0, ichunk += 4, ibuf = ibuf == scales0 + 2 * CHUNK_BYTES ? scales0 : ibuf + CHUNK_BYTES;
    };
    // K ends inside the last block: pieces behind it come from the weight's own padding, which is zero there (a piece of
    // 16 behind K exists in the first tile's last block, its very last)
    const bool ragged = p.K % 128 != 0;
    const uint8_t* const zeros = p.w + (int64_t)(p.G - 1) * 2048 + 1024 + 48 * 16;
    const int KT = (p.G - 1) / KS + 1;  // (in the last stage of an odd number of blocks the second group repeats the last, times 0)
    // transfer t of stage st into the buffer at LDS address `at`
    auto dma = [&](auto tc, auto fullc, int st, uint32_t at) {
        constexpr int t = decltype(tc)::value;
        constexpr bool FULL = decltype(fullc)::value;  // the stage is known to be whole blocks of K
        const int blk = FULL ? st * KS + group : min(st * KS + group, p.G - 1);
        if constexpr (t < DX) {
            const uint32_t m0v = at + (uint32_t)(wave * DX + t) * 1024;
            if (!FULL && ragged && blk == p.G - 1) {
                const uint8_t* a = blk * 128 + xk[t] < p.K ? xbase + xoff[t] + (int64_t)blk * 128 : zeros;
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(m0v), "v"(a) : "memory");
            } else {
                const uint8_t* s = xbase + (int64_t)blk * 128;
                const uint32_t o = xoff[t];
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0v), "v"(o), "s"(s) : "memory");
            }
        } else {
            constexpr int u = t - DX;
            const uint32_t m0v = at + XB + (uint32_t)(wave * DW + u) * 1024;
            const uint8_t* s = wtile[u / 2] + (int64_t)blk * 2048 + (u & 1) * 1024;
            const uint32_t o = woff;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0v), "v"(o), "s"(s) : "memory");
        }
    };
    // Everything this wavefront has requested has landed but for its last `keep` transfers (they land in the order of
    // issue; the scaling wavefronts' scales are not counted, so that they wait for one transfer or two more), and so for
    // all wavefronts behind the barrier.
    auto landed = [&](auto keepc) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(keepc)::value) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    using std::integral_constant;
    using none = integral_constant<int, 0>;

    // ---- fragments: lane l supplies bytes 16 c .. 16 c + 15 of both halves of row l % 16, c = l / 16
    const int r = lane & 15, c = lane >> 4;
    const uint32_t fx0 = (uint32_t)((wm * 16 * TI + r) * 128 + (c ^ swz(r)) * 16);
    const uint32_t fx1 = (uint32_t)((wm * 16 * TI + r) * 128 + ((4 + c) ^ swz(r)) * 16);
    const uint32_t fw = (uint32_t)(XB + wn * TJ * 2048 + lane * 16);
    const uint32_t fs = scales0 + (wm * 16 * TI + r) * 16, fsw = scales0 + BM * 16 + (wn * 16 * TJ / 128) * 16;
    i32x4 xf[TI][2], wf[2][2][2];  // token fragments; channel fragments of two pairs
    float sx[TI], sw;
    auto read_x = [&](int i, uint32_t at) {
        xf[i][0] = *reinterpret_cast<const i32x4*>(lds + at + fx0 + i * 2048);
        xf[i][1] = *reinterpret_cast<const i32x4*>(lds + at + fx1 + i * 2048);
    };
    auto read_w = [&](int set, int pair, uint32_t at) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                wf[set][h][e] = *reinterpret_cast<const i32x4*>(lds + at + fw + (2 * pair + h) * 2048 + e * 1024);
    };
    uint32_t so = 0;  // where the next stage's scales lie
    auto read_s = [&]() {
#pragma unroll
        for (int i = 0; i < TI; i++) sx[i] = *reinterpret_cast<const float*>(lds + so + fs + i * 256);
        sw = *reinterpret_cast<const float*>(lds + so + fsw);
        so += 4;
        if ((so & 15) == 0) so = so == 2 * CHUNK_BYTES + 16 ? 0 : so + CHUNK_BYTES - 16;
    };
    static_assert(CHUNK_BYTES % 16 == 0, "read_s counts by it");

    f32x4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; i++)
#pragma unroll
        for (int j = 0; j < TJ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // One stage, in pairs of channel fragments, token fragment by token fragment within a pair.  While a pair is multiplied
    // the next one is read.  The last pair starts with the stage's barrier: everything of this stage has been read by then
    // and the next one has landed, so the last pair reads the next stage's first fragments, a token fragment as soon as
    // its last product is issued.  A product's four results meet their scale two products later, when the matrix core has
    // long delivered them.
    //
    // The transfers stand between the products, spread out: the CU's address unit takes about 22 cycles for each, and a
    // wavefront that finds it busy waits with its products behind it (all of a stage's in its last pair: 2 us of 52 on 128
    // workgroups of 256 x 256).  With three buffers and more, stage st requests stage st + NB - 1 into the buffer that the
    // last barrier freed.  With two, that would leave a stage's last transfers no time to land; there the two halves of
    // the buffer are freed one after the other: the x half by a barrier behind the first pair (the token fragments are in
    // registers by then), refilled during the middle pairs, the w half by the stage's own barrier, refilled during its
    // last pair and the next one's first.
    constexpr int Q = TI * TJ, QB = Q - 2 * TI;  // products of a stage; the first one behind its barrier
    constexpr int T = DX + DW;
    constexpr int AHEAD = NB >= 3 ? NB - 1 : 2;  // stages requested before the first
    f32x4 late[2] = {};  // the results of the stage's last two products, settled behind the next stage's first two
    float late_s = 0.0f;
    auto settle_into = [&](int q, const f32x4& d, float s) {
        auto& a = acc[q / 2 % TI][2 * (q / (2 * TI)) + q % 2];
#pragma unroll
        for (int t = 0; t < 4; t++) a[t] = fmaf(d[t], s, a[t]);
        // (here and not later: left alone, the compiler gathers a stage's multiply-adds behind its last product, with every
        // product's result kept until then)
        asm volatile("" : "+v"(a));
    };
    // KIND 0: what it requests exists and is a whole block of K (no branches); 1: any stage but the last; 2: the last
    auto stage = [&](auto kindc, int st, uint32_t at, uint32_t next, uint32_t prev) {
        constexpr int KIND = decltype(kindc)::value;
        constexpr bool LAST = KIND == 2;
        using full = integral_constant<bool, KIND == 0>;
        const bool more = KIND == 0 || st + AHEAD < KT;
        float s[TI];
        f32x4 part[3];
        auto settle = [&](auto qc) {  // product q of the stage: pair q / (2 TI), token (q / 2) % TI, half q % 2
            constexpr int q = decltype(qc)::value;
            if constexpr (q < 0)
                settle_into(Q + q, late[2 + q], late_s);
            else
                settle_into(q, part[q % 3], s[q / 2 % TI]);
        };
        auto transfers = [&](auto qc) {  // behind product q
            constexpr int q = decltype(qc)::value;
            auto some = [&](auto firstc, auto endc, int to, uint32_t buffer) {
                constexpr int first = decltype(firstc)::value, end = decltype(endc)::value;
                static_for<end - first>([&](auto d) { dma(integral_constant<int, first + decltype(d)::value>{}, full{}, to, lds0 + buffer); });
            };
            if constexpr (LAST) {
            } else if constexpr (NB >= 3) {
                constexpr int from = q * T / Q, to = (q + 1) * T / Q;
                if constexpr (to > from)
                    if (more) some(integral_constant<int, from>{}, integral_constant<int, to>{}, st + NB - 1, prev);
                if constexpr (q == Q - 1)
                    if (more) next_scales();
            } else {
                constexpr int HALF = DW / 2, FIRST = 2 * TI;  // products of the first pair, and of the last
                if constexpr (q < FIRST) {
                    constexpr int from = DX + HALF + q * (DW - HALF) / FIRST, to = DX + HALF + (q + 1) * (DW - HALF) / FIRST;
                    if constexpr (to > from)
                        some(integral_constant<int, from>{}, integral_constant<int, to>{}, st + 1, next);
                } else if constexpr (q < QB) {
                    constexpr int from = (q - FIRST) * DX / (QB - FIRST), to = (q - FIRST + 1) * DX / (QB - FIRST);
                    if constexpr (to > from)
                        if (more) some(integral_constant<int, from>{}, integral_constant<int, to>{}, st + 2, at);
                    if constexpr (q == QB - 1)
                        if (more) next_scales();
                } else {
                    constexpr int from = DX + (q - QB) * HALF / FIRST, to = DX + (q - QB + 1) * HALF / FIRST;
                    if constexpr (to > from)
                        if (more) some(integral_constant<int, from>{}, integral_constant<int, to>{}, st + 2, at);
                }
            }
        };
        static_for<PAIRS>([&](auto pc) {
            constexpr int pr = decltype(pc)::value;
            constexpr bool END = pr == PAIRS - 1;
            if constexpr (pr == 0) {
#pragma unroll
                for (int i = 0; i < TI; i++) s[i] = KS > 1 && LAST && st * KS + group >= p.G ? 0.0f : sx[i] * sw;
            }
            if constexpr (NB == 2 && pr == 1 && !LAST) {
                if (more) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wavefront's token fragments are in registers
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
            }
            if constexpr (!END)
                read_w((pr + 1) & 1, pr + 1, at);
            else if constexpr (!LAST) {
                // under way may be: what this stage has requested so far, and (four buffers) the stage after the next one
                if constexpr (NB >= 3) {
                    if (more)
                        landed(integral_constant<int, (NB - 3) * T + QB * T / Q>{});
                    else if (NB == 4 && st + 2 < KT)
                        landed(integral_constant<int, T>{});
                    else
                        landed(none{});
                } else {
                    if (more)
                        landed(integral_constant<int, DX>{});
                    else
                        landed(none{});
                }
                read_w((pr + 1) & 1, 0, next);
                read_s();
            }
            __builtin_amdgcn_sched_barrier(0);
            const Operand<EXACT> w0(wf[pr & 1][0][0], wf[pr & 1][0][1]), w1(wf[pr & 1][1][0], wf[pr & 1][1][1]);
            static_for<TI>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                constexpr int q = (pr * TI + i) * 2;
                const Operand<EXACT> x(xf[i][0], xf[i][1]);
                part[q % 3] = block_sum(w0, x);
                __builtin_amdgcn_sched_barrier(0);
                settle(integral_constant<int, q - 2>{});
                transfers(integral_constant<int, q>{});
                __builtin_amdgcn_sched_barrier(0);
                part[(q + 1) % 3] = block_sum(w1, x);
                __builtin_amdgcn_sched_barrier(0);
                settle(integral_constant<int, q - 1>{});
                if constexpr (END && !LAST) read_x(i, next);
                transfers(integral_constant<int, q + 1>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        late[0] = part[(Q - 2) % 3], late[1] = part[(Q - 1) % 3], late_s = s[TI - 1];
    };

    if (scaling)
        for (int q = 0; q < 4; q++) scale_dma(q, 0, scales0);
    // (two buffers: the second half of stage 1's weights follows in stage 0, as in every stage)
    constexpr int SECOND = NB >= 3 ? T : DX + DW / 2;
    for (int st = 0; st < min(AHEAD, KT); st++) {
        if (NB >= 3 || st == 0)
            static_for<T>([&](auto t) { dma(t, std::false_type{}, st, lds0 + st * STAGE); });
        else
            static_for<SECOND>([&](auto t) { dma(t, std::false_type{}, st, lds0 + st * STAGE); });
        next_scales();
    }
    if (KT >= AHEAD)
        landed(integral_constant<int, (AHEAD - 1) * SECOND>{});
    else
        landed(none{});
    // (a wait that the compiler sees: it would otherwise hold scalar loads of the kernel's arguments for possibly under way
    // and, since those return in any order, wait for every LDS read at the head of each stage)
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    read_w(0, 0, 0);
    read_s();
#pragma unroll
    for (int i = 0; i < TI; i++) read_x(i, 0);
    uint32_t at = 0, prev = (NB - 1) * STAGE;
    int st = 0;
    auto walk = [&](auto kindc, int end) {
        for (; st < end; st++) {
            const uint32_t next = at == (NB - 1) * STAGE ? 0 : at + STAGE;
            stage(kindc, st, at, next, prev);
            prev = at, at = next;
        }
    };
    walk(integral_constant<int, 0>{}, (ragged ? p.G - 1 : p.G) / KS - AHEAD);
    walk(integral_constant<int, 1>{}, KT - 1);
    stage(integral_constant<int, 2>{}, KT - 1, at, 0, 0);
    settle_into(Q - 2, late[0], late_s);
    settle_into(Q - 1, late[1], late_s);
    // (the bias is requested here, all of a lane's channels at once, into the registers that the fragments leave; a fragment at
    // a time in the passes below, 1024 rows over 4096 -> 4096 took 23.5 us instead of 23.1)
    float b[TJ][4];
#pragma unroll
    for (int j = 0; j < TJ; j++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int n = min(n0 + wn * 16 * TJ + 16 * j + 4 * c + t, p.N - 1);
            b[j][t] = 0.0f;
            if (p.bias)
                b[j][t] = p.bias_dtype == NQ_DT_F32 ? reinterpret_cast<const float*>(p.bias)[n]
                                                    : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p.bias)[n] << 16);
        }
    __syncthreads();  // (nothing is under way: the last requests were waited for a stage ago)
    if constexpr (KS == 2) {
        static_assert(WAVES * TI * TJ * 1024 <= GROUP, "the second group's results in its own LDS");
        f32x4* const meet = reinterpret_cast<f32x4*>(lds_all + GROUP) + wave * TI * TJ * 64 + lane;
        if (group == 1) {
#pragma unroll
            for (int q = 0; q < TI * TJ; q++) meet[q * 64] = acc[q / TJ][q % TJ];
        }
        __syncthreads();
        if (group == 1) return;
#pragma unroll
        for (int q = 0; q < TI * TJ; q++) acc[q / TJ][q % TJ] += meet[q * 64];
    }

    // ---- epilogue: a lane holds token 16 i + r and channels 16 j + 4 c .. + 3.  A wavefront stages 32 tokens at a time in
    // LDS of its own and writes them as 128-bit stores, whole rows of its channels.
    constexpr int ES = EXACT ? 4 : 2, CH = 16 * TJ, ROWB = CH * ES + 16;
    static_assert(WAVES * 32 * ROWB <= NB * STAGE, "the epilogue stages in the stage buffers");
    uint8_t* const stg = lds + wave * 32 * ROWB;
    const int wm0 = m0 + wm * 16 * TI, wn0 = n0 + wn * CH;
    // (a row-fused layer's parts begin on blocks of 128 channels, so all of a wavefront's lie in one, and a fused call is one
    // launch: 1024 rows over 4096 -> 4096 | 1024 | 1024 in bf16 30.9 us, part by part 58.8)
    void* part_y;
    int width, col;
    seg_lookup(p.seg, wn0, part_y, width, col);
    uint8_t* const y = reinterpret_cast<uint8_t*>(part_y);
    const bool whole = col + CH <= width && width % (16 / ES) == 0 && ((uintptr_t)y & 15) == 0;
#pragma unroll
    for (int ip = 0; ip < TI; ip += 2) {
#pragma unroll
        for (int j = 0; j < TJ; j++) {
#pragma unroll
            for (int ii = 0; ii < 2; ii++) {
                f32x4 z;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    z[t] = acc[ip + ii][j][t] + b[j][t];
                    if (p.relu) z[t] = z[t] > 0.0f ? z[t] : 0.0f;
                }
                uint8_t* dst = stg + (16 * ii + r) * ROWB + (16 * j + 4 * c) * ES;
                if constexpr (EXACT)
                    *reinterpret_cast<f32x4*>(dst) = z;
                else
                    *reinterpret_cast<bf16x4*>(dst) = __builtin_convertvector(z, bf16x4);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (whole) {
            constexpr int LPR = CH * ES / 16, RPI = 64 / LPR;  // lanes per row, rows per instruction
#pragma unroll
            for (int t = 0; t < 32 / RPI; t++) {
                const int row = t * RPI + lane / LPR, c16 = lane % LPR;
                const i32x4 v = *reinterpret_cast<const i32x4*>(stg + row * ROWB + c16 * 16);
                const int m = wm0 + 16 * ip + row, n = col + c16 * (16 / ES);
                if (m < p.M) *reinterpret_cast<i32x4*>(y + ((int64_t)m * width + n) * ES) = v;
            }
        } else if (width > col) {
            // rows that do not begin on 16 bytes, or end inside the tile: 4 bytes per lane, adjacent lanes adjacent (bf16 rows
            // that begin on an odd element: pairs from the second one on, and the ends alone).  Every row's loads and stores without
            // a branch: 1024 rows over 960 -> 2567 in bf16 10.2 us, with a loop of its own per row 14.6, 2560 channels 9.0
            const int limit = min(CH, width - col);
            if constexpr (EXACT) {
                static_assert(CH == 64, "a row per instruction");
#pragma unroll 8
                for (int row = 0; row < 32; row++) {
                    const int m = wm0 + 16 * ip + row;
                    const float v = reinterpret_cast<const float*>(stg + row * ROWB)[lane];
                    if (m < p.M && lane < limit) reinterpret_cast<float*>(y)[(int64_t)m * width + col + lane] = v;
                }
            } else {
                constexpr int LPR = CH / 2, RPI = 64 / LPR;
                const int j = lane % LPR, m = wm0 + 16 * ip + lane / LPR;
                uint16_t* const d = reinterpret_cast<uint16_t*>(y) + (int64_t)m * width + col;
                const uint32_t* src = reinterpret_cast<const uint32_t*>(stg + lane / LPR * ROWB) + j;
#pragma unroll 8
                for (int t = 0; t < 32 / RPI; t++) {
                    const uint32_t w0 = src[t * RPI * ROWB / 4], w1 = src[t * RPI * ROWB / 4 + 1];  // (16 spare bytes behind a row)
                    const int odd = (int)((uintptr_t)d / 2 + t * RPI * width) & 1, e = 2 * j + odd;
                    if (m + t * RPI < p.M && e + 1 < limit)
                        *reinterpret_cast<uint32_t*>(d + (int64_t)t * RPI * width + e) = odd ? w0 >> 16 | w1 << 16 : w0;
                }
                // the ends alone: lanes 2 r and 2 r + 1 look after row r's first and last element
                const int r1 = lane / 2, end = lane & 1 ? limit - 1 : 0;
                uint16_t* const d1 = reinterpret_cast<uint16_t*>(y) + (int64_t)(wm0 + 16 * ip + r1) * width + col;
                const int odd1 = (int)((uintptr_t)d1 / 2) & 1;
                if (wm0 + 16 * ip + r1 < p.M && (lane & 1 ? (limit - odd1) & 1 : odd1))
                    d1[end] = reinterpret_cast<const uint16_t*>(stg + r1 * ROWB)[end];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

template <int BM, int BN, int NB, int KS>
constexpr size_t lds_bytes() { return KS * ((size_t)NB * (BM + BN) * 128 + 3 * (BM * 16 + 256)); }

template <int BM, int BN, int WM, int WN, int NB, int KS, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN * KS) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp8_block_gemm_kernel(const BlockParams p) {
    block_gemm_body<BM, BN, WM, WN, NB, KS, EXACT>(p);
}

// `grid`: the first that many tiles of the order only (0: all of the region from m_base, n_base on)
template <int BM, int BN, int WM, int WN, int NB, int KS, bool EXACT>
int32_t launch(BlockParams p, hipStream_t s, int64_t grid = 0) {
    static LdsAttrOnce attr;
    p.tiles_m = (p.M - p.m_base - 1) / BM + 1, p.tiles_n = (p.N - p.n_base - 1) / BN + 1;
    if (grid == 0) grid = (int64_t)p.tiles_m * p.tiles_n;  // (fits a launch: pick)
    const void* kernel = reinterpret_cast<const void*>(&fp8_block_gemm_kernel<BM, BN, WM, WN, NB, KS, EXACT>);
    NQ_HIP(set_max_lds_once(attr, kernel, lds_bytes<BM, BN, NB, KS>()));
    hipLaunchKernelGGL((fp8_block_gemm_kernel<BM, BN, WM, WN, NB, KS, EXACT>), dim3((unsigned)grid), dim3(64 * WM * WN * KS), (lds_bytes<BM, BN, NB, KS>()), s, p);
    NQ_HIP(hipGetLastError());
    return NQ_OK;
}

// What a call takes on each tile, in microseconds: rounds of as many workgroups as the chip holds, each a fixed part and a
// part per block of K, which lengthens as more CUs draw on L2 (`crowd`: from 0 at `from` workgroups to 1 at `full`).
// Measured over M = 256 .. 8192, K = 960 and 4096, N = 960 .. 11008 (K = 4096, N = 4096; M = 256 / 512 / 1024 / 2048 / 4096):
//   bf16 y   128 x 128: 18.2 / 18.5 / 20.6 / 44.6 / 89     128 x 256: 26.7 / 27.0 / 27.7 / 35.8 / 71
//            256 x 256: 46.5 / 46.8 / 47.1 / 50.1 / 60.4
//             64 x 128, K dealt over two groups: 15.3 / 16.0 / 29.5 / - / -
//   fp32 y    64 x 128: 26.0 / 26.6 / 39.6 / 77 / 153      128 x 128: 33.7 / 34.5 / 36.8 / 72 / 141
//            256 x 128: 54.1 / 54.8 / 56.6 / 61.5 / 120     64 x 128, two groups: 20.9 / 22.2 / 40.5 / - / -
// (Two groups of four wavefronts: alone on its SIMD a wavefront's multiply-adds stand in the way of its products; two share it,
// each with a block of its own.  Only 64 x 128 tiles leave room in LDS for two groups' three buffers.)
struct Form {
    int bm, bn;
    double fixed, step, crowd;
    int from, full;
};
constexpr Form F256{256, 256, 8.0, 1.20, 0.40, 64, 256}, F128x256{128, 256, 5.8, 0.665, 0.275, 128, 256},
    F128{128, 128, 4.5, 0.44, 0.06, 128, 256}, F64K2{64, 128, 4.2, 0.36, 0.02, 128, 256},
    E256x128{256, 128, 6.5, 1.52, 0.20, 64, 256}, E128{128, 128, 4.5, 0.92, 0.09, 128, 256},
    E64{64, 128, 4.5, 0.69, 0.41, 256, 512}, E64K2{64, 128, 5.5, 0.485, 0.04, 128, 256};

// `off`: what rows off 16 bytes cost per 64 x 32 results of a wavefront (the last stores of the kernel: 1.2 us in bf16, 0.5 in fp32)
double estimate(const Form& f, int64_t workgroups, int G, double off) {
    const int64_t rounds = (workgroups + f.full - 1) / f.full;
    const double in_round = (double)workgroups / (double)rounds;
    const double crowd = in_round > f.from ? (in_round - f.from) / (double)(f.full - f.from) : 0.0;
    return (double)rounds * (f.fixed + off * std::max(1, f.bm * f.bn / 16384) + G * (f.step + f.crowd * crowd));
}
double estimate(const Form& f, int M, int N, int G, double off) {
    return estimate(f, (int64_t)((M - 1) / f.bm + 1) * ((N - 1) / f.bn + 1), G, off);
}

// The 256 x 256 tiles that do not fill a round of 256 workgroups go on 128 x 256 tiles in a second launch, where they are
// at most half a round and whole columns of the last band of 8 row tiles (M = 8192, N = 11008: 96 of 1376, 12 columns).
// Every result adds the same blocks in the same order on any tile: same bits.
int64_t leftover(int M, int N) {
    const int64_t tm = (M - 1) / 256 + 1, tn = (N - 1) / 256 + 1, rest = tm * tn % 256, rows = tm - (tm - 1) / 8 * 8;
    return tm * tn > 256 && rest > 0 && rest <= 128 && rest % rows == 0 && rest / rows <= tn ? rest : 0;
}
double estimate256(int M, int N, int G, double off) {
    const int64_t tiles = (int64_t)((M - 1) / 256 + 1) * ((N - 1) / 256 + 1), rest = leftover(M, N);
    return rest ? estimate(F256, tiles - rest, G, off) + estimate(F128x256, 2 * rest, G, off) : estimate(F256, tiles, G, off);
}

// the form of lowest estimate among those whose launch has fewer than 2^31 threads, and that estimate; null where none has,
// or a tile's rows are beyond 32-bit offsets from its base
const Form* pick(const BlockParams& p, double* us) {
    if (p.M <= 64 || (int64_t)p.K * 256 >= ((int64_t)1 << 32)) return nullptr;
    const bool exact = p.y_dtype == NQ_DT_F32;
    const double off = p.N % (exact ? 4 : 8) == 0 ? 0.0 : exact ? 0.5 : 1.2;
    const Form* best = nullptr;
    const auto consider = [&](const Form& f) {
        if ((int64_t)((p.M - 1) / f.bm + 1) * ((p.N - 1) / f.bn + 1) * 512 > INT32_MAX) return;
        const double t = &f == &F256 ? estimate256(p.M, p.N, p.G, off) : estimate(f, p.M, p.N, p.G, off);
        if (!best || t < *us) *us = t, best = &f;
    };
    if (exact)
        consider(E256x128), consider(E128), consider(E64), consider(E64K2);
    else
        consider(F256), consider(F128x256), consider(F128), consider(F64K2);
    return best;
}

}  // namespace

bool fp8_block_gemm_estimate_us(const BlockParams& p, double* us) { return pick(p, us) != nullptr; }

void fp8_block_gemm_form(const BlockParams& p, int32_t* form) {
    double us;
    const Form* f = pick(p, &us);
    form[0] = 1, form[1] = f->bm, form[2] = f->bn, form[3] = f == &E64K2 || f == &F64K2 ? 2 : 1;
    form[4] = f == &F256 ? (int32_t)leftover(p.M, p.N) : 0;
}

int32_t launch_fp8_block_gemm(const BlockParams& p, hipStream_t s) {
    double us;
    const Form* f = pick(p, &us);
    if (f == &E64) return launch<64, 128, 2, 2, 3, 1, true>(p, s);
    if (f == &E64K2) return launch<64, 128, 2, 2, 3, 2, true>(p, s);
    if (f == &E128) return launch<128, 128, 4, 2, 4, 1, true>(p, s);
    if (f == &E256x128) return launch<256, 128, 4, 2, 3, 1, true>(p, s);
    if (f == &F64K2) return launch<64, 128, 2, 2, 3, 2, false>(p, s);
    if (f == &F128) return launch<128, 128, 4, 2, 4, 1, false>(p, s);
    if (f == &F128x256) return launch<128, 256, 4, 2, 3, 1, false>(p, s);
    const int64_t rest = leftover(p.M, p.N);
    if (!rest) return launch<256, 256, 4, 2, 2, 1, false>(p, s);
    const int tm = (p.M - 1) / 256 + 1, tn = (p.N - 1) / 256 + 1, rows = tm - (tm - 1) / 8 * 8;
    const int32_t rc = launch<256, 256, 4, 2, 2, 1, false>(p, s, (int64_t)tm * tn - rest);
    if (rc) return rc;
    BlockParams q = p;
    q.m_base = (tm - rows) * 256, q.n_base = (tn - (int)(rest / rows)) * 256;
    return launch<128, 256, 4, 2, 3, 1, false>(q, s);
}

}  // namespace nq
