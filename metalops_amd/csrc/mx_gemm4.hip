// Y[M, N] = X[M, K] W[N, K]^T, both operands MXFP4, through LDS, for many rows.
//
// v_mfma_scale_f32_32x32x64 multiplies packed blocks as they stand: lane l of an operand holds
// one block (16 bytes) of row l % 32 and its scale byte, 64 elements of K a step, at four times
// the rate of 16-bit operands.  So the kernel is bound by feeding it: a workgroup of four waves
// (2 x 2) computes 64 TM rows x 64 TN columns, a wave 32 TM x 32 TN, and a stage is 128
// elements of K, four blocks, of which lane half h = l / 32 takes blocks 2 h and 2 h + 1 (the
// order of K is free as long as both operands keep it).
//
// LDS holds four stages; a row's 16-byte chunk c lies at c ^ (row / 4) % 4, so that 16 lanes
// reading one chunk of 16 rows meet 16 banks.  Copies go out three stages ahead, between the
// MFMAs, as do the LDS reads of the next step; one barrier a stage.  Scales are copied 16 bytes
// a row at a time, the aligned pieces that hold a row's bytes, for four stages.  A row's four
// bytes of a stage lie in two neighbouring dwords (rows of any length: K / 32 need not be a
// multiple of 4), from which one 64-bit shift takes the lane's two.
//
// 2048 x 4096 x 14336 takes 79 us (3.0 PFLOP/s), the matrix cores 40% busy: the 448 tiles of
// 256 x 256 are two rounds of 256 workgroups, the second not full, and a tile's 32 stages are
// short beside its start and its stores, which nothing overlaps at one workgroup a CU (LDS and
// registers hold no second one; tiles of 128 x 128, which would, read twice as much and take 107).
#include <algorithm>
#include <type_traits>

#include "mx_gemm.h"

namespace mcq4 {

struct MxGemm4Args {
    const uint8_t *X, *Xs, *W, *Ws;
    void *Y;
    int64_t ldy;
    int M, nb, N;
    int stages, tiles_m, S;
    float *part;
    int64_t ldp;
};

template <int TM, int TN>
struct MxGemm4Lds {
    static constexpr int ROWS = 64 * (TM + TN);                  // X's rows, then W's
    static constexpr int SLOT = ROWS * 64, S_SLOT = ROWS * 16, S0 = 4 * SLOT, LOOP = S0 + 3 * S_SLOT;
    template <int YT>
    static constexpr int total() { return std::max(LOOP, 4 * mx_store_lds<YT, TM, TN>()); }
};

template <int YT, int TM, int TN>
__global__ void __launch_bounds__(256, TM * TN >= 16 ? 1 : 2)
mx_gemm4_kernel(MxGemm4Args a) {
    typedef MxGemm4Lds<TM, TN> L;
    constexpr int BM = 64 * TM, BN = 64 * TN;
    constexpr int NX = TM, NW = TN;                      // copies of a wave and stage: 16 rows each
    constexpr int NMF = TM * TN;                         // MFMAs of a step
    static_assert((TM + TN) % 4 == 0, "each wave copies as many scales");
    constexpr int NS = (TM + TN) / 4;                    // copies of scales: 64 rows each
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lrow = lane & 31, lhi = lane >> 5;
    const int wm = (wave & 1) * 32 * TM, wn = (wave >> 1) * 32 * TN;        // this wave's rows and columns
    const MxTile tile = mx_tile(a.tiles_m);
    const int m0 = tile.m * BM, n0 = tile.n * BN;
    const int s0 = (int)((uint32_t)a.stages * blockIdx.z / (uint32_t)a.S), s1 = (int)((uint32_t)a.stages * (blockIdx.z + 1) / (uint32_t)a.S);
    const int nk = min(4 * s1, a.nb) - 4 * s0;           // blocks
    const int nst = s1 - s0, nfull = nk >> 2;

    const uint32_t lds0 = lds_addr(smem);
    const int row = a.nb * 16;
    const int rows_m = min(a.M - m0, BM), rows_n = min(a.N - n0, BN);
    const uint8_t *x_base = a.X + (int64_t)m0 * row + (int64_t)s0 * 64, *w_base = a.W + (int64_t)n0 * row + (int64_t)s0 * 64;
    const int x_bytes = rows_m * row - s0 * 64, w_bytes = rows_n * row - s0 * 64;
    const int vo_c = (lane >> 2) * row + 16 * ((lane ^ (lane >> 4)) & 3);
    auto copy = [&](int s, int ci) {
        const int off = 64 * min(s, nst - 1);
        uint8_t *const slot = smem + (s & 3) * L::SLOT;
        if (ci < NX) {
            const int r = 16 * (wave * NX + ci);
            mx_copy16(mx_rsrc(x_base + off, x_bytes - off), slot + 64 * r, vo_c + r * row, 0);
        } else {
            const int r = 16 * (wave * NW + ci - NX);
            mx_copy16(mx_rsrc(w_base + off, w_bytes - off), slot + 64 * (BM + r), vo_c + r * row, 0);
        }
    };
    // Scales: from the aligned dword of the tile's first byte on.  Piece g of a row: its
    // aligned dwords 4 g .. 4 g + 3 (of this split).  Wave w copies 64-row groups w, w + 4.
    const uint8_t *xs_first = a.Xs + (int64_t)m0 * a.nb + 4 * s0, *ws_first = a.Ws + (int64_t)n0 * a.nb + 4 * s0;
    const int x_ph = (int)((uintptr_t)xs_first & 3), w_ph = (int)((uintptr_t)ws_first & 3);
    const int xs_bytes = (x_ph + rows_m * a.nb - 4 * s0 + 3) & ~3, ws_bytes = (w_ph + rows_n * a.nb - 4 * s0 + 3) & ~3;
    auto copy_s = [&](int g, int slot, int ci) {
        const int grp = wave + 4 * ci, off = 16 * g;                 // TM + TN is a multiple of four
        const bool is_x = grp < TM;
        const uint8_t *base = is_x ? xs_first - x_ph : ws_first - w_ph;
        const int vo = is_x ? x_ph + (64 * grp + lane) * a.nb : w_ph + (64 * (grp - TM) + lane) * a.nb;
        mx_copy16(mx_rsrc(base + off, (is_x ? xs_bytes : ws_bytes) - off), smem + L::S0 + slot * L::S_SLOT + grp * 1024, vo & ~3, 0);
    };

    uint32_t d_off[2];                                   // chunk 2 h + t of row l % 32
#pragma unroll
    for (int t = 0; t < 2; ++t) d_off[t] = lds0 + lrow * 64 + (((2 * lhi + t) ^ ((lrow >> 2) & 3)) << 4);
    auto read_x = [&](int s, int t, int i) { return mx_lds16(d_off[t] + (s & 3) * L::SLOT + (wm + 32 * i) * 64); };
    auto read_w = [&](int s, int t, int j) { return mx_lds16(d_off[t] + (s & 3) * L::SLOT + (BM + wn + 32 * j) * 64); };
    // Dword d of a row's scales, and where in a pair of them the lane's two bytes start.
    int g_slot = 0;                                      // slot of piece (d / 4) for the dwords read now
    auto read_s = [&](int d, int r) { return mx_lds4(lds0 + L::S0 + g_slot * L::S_SLOT + (r + lrow) * 16 + 4 * (d & 3)); };
    uint32_t sh_x[TM], sh_w[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) sh_x[i] = 8 * (((x_ph + (wm + 32 * i + lrow) * a.nb) & 3) + 2 * lhi);
#pragma unroll
    for (int j = 0; j < TN; ++j) sh_w[j] = 8 * (((w_ph + (wn + 32 * j + lrow) * a.nb) & 3) + 2 * lhi);
    auto pick = [&](uint32_t lo, uint32_t hi, uint32_t sh) { return (uint32_t)((((uint64_t)hi << 32) | lo) >> sh); };

    float16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    struct Step { uint4_t x[TM], w[TN]; };
    struct Scales { uint32_t x[TM], w[TN]; };
    Step A, B;
    Scales now, lo, hi;                                  // this stage's bytes; dwords s + 1 and s + 2 of the rows

    auto mfma = [&](auto t, int i, int j, const Step &o) {
        constexpr int T = decltype(t)::value;
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(o.w[j]), mx_operand(o.x[i]), acc[i][j], 4, 4,
                                                                    T, (int)now.w[j], T, (int)now.x[i]);
    };
    typedef std::integral_constant<int, 0> t0;
    typedef std::integral_constant<int, 1> t1;
    // Both steps read the next step's operands between their MFMAs.  Step 0 also sends out the
    // copies and reads dword s + 2 of the scales; step 1 ends with the next stage's bytes.
    auto step0 = [&](int s) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int idx = 0; idx < NMF; ++idx) {
            const int i = idx / TN, j = idx % TN;
            mfma(t0{}, i, j, A);
#pragma unroll
            for (int c = 0; c < TM + TN; ++c) {
                if (c * NMF / 2 / (TM + TN) == idx) {
                    if (c < TM) B.x[c] = read_x(s, 1, c);
                    else B.w[c - TM] = read_w(s, 1, c - TM);
                }
                if (NMF / 2 + c * NMF / 2 / (TM + TN) == idx) {
                    if (c < TM) hi.x[c] = read_s(s + 2, wm + 32 * c);
                    else hi.w[c - TM] = read_s(s + 2, BM + wn + 32 * (c - TM));
                }
                if (c * NMF / (TM + TN) == idx) copy(s + 3, c);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto step1 = [&](int s) {
        Scales next;
#pragma unroll
        for (int idx = 0; idx < NMF; ++idx) {
            const int i = idx / TN, j = idx % TN;
            mfma(t1{}, i, j, B);
#pragma unroll
            for (int c = 0; c < TM + TN; ++c) {
                if (c * NMF / 2 / (TM + TN) == idx) {
                    if (c < TM) A.x[c] = read_x(s + 1, 0, c);
                    else A.w[c - TM] = read_w(s + 1, 0, c - TM);
                }
                if (NMF / 2 + c * NMF / 2 / (TM + TN) == idx) {
                    if (c < TM) {
                        next.x[c] = pick(lo.x[c], hi.x[c], sh_x[c]);
                        lo.x[c] = hi.x[c];
                    } else {
                        next.w[c - TM] = pick(lo.w[c - TM], hi.w[c - TM], sh_w[c - TM]);
                        lo.w[c - TM] = hi.w[c - TM];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        now = next;
    };

#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int c = 0; c < NS; ++c) copy_s(g, g, c);
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int c = 0; c < NX + NW; ++c) copy(s, c);
    wait_vmcnt<NX + NW>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        A.x[i] = read_x(0, 0, i);
        const uint32_t d0 = read_s(0, wm + 32 * i);
        lo.x[i] = read_s(1, wm + 32 * i);
        now.x[i] = pick(d0, lo.x[i], sh_x[i]);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        A.w[j] = read_w(0, 0, j);
        const uint32_t d0 = read_s(0, BM + wn + 32 * j);
        lo.w[j] = read_s(1, BM + wn + 32 * j);
        now.w[j] = pick(d0, lo.w[j], sh_w[j]);
    }
    // The barrier before a stage makes the next one visible and ends every wave's reads of the one
    // before, whose slot this stage's copies fill.  Scale piece g is sent out in stage 4 g - 8,
    // ahead of that stage's other copies, and first read in stage 4 g - 2.
    int g0 = 0, g1 = 1, g2 = 2;                          // slots of pieces s / 4, the next, the one after
    for (int s = 0; s < nfull; ++s) {
        if (s > 0) {
            wait_vmcnt<NX + NW>();
            lds_barrier();
        }
        if ((s & 3) == 0) {
            if (s > 0) { const int t = g0; g0 = g1; g1 = g2; g2 = t; }
#pragma unroll
            for (int c = 0; c < NS; ++c) copy_s((s >> 2) + 2, g2, c);
        }
        g_slot = (s & 3) >= 2 ? g1 : g0;                 // dword s + 2
        step0(s);
        step1(s);
    }
    wait_vmcnt<0>();
    lds_barrier();
    if (nk & 3) {
        // One to three blocks left: the others' codes and scales are what lies behind the row.
        const int left = nk & 3;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const bool in = 2 * lhi + t < left;
            Step o;
            Scales sc;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                o.x[i] = read_x(nfull, t, i);
                if (!in) o.x[i] = uint4_t{0, 0, 0, 0};
                sc.x[i] = in ? now.x[i] >> (8 * t) : 0u;
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                o.w[j] = read_w(nfull, t, j);
                sc.w[j] = in ? now.w[j] >> (8 * t) : 0u;
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(o.w[j]), mx_operand(o.x[i]), acc[i][j], 4, 4,
                                                                                0, (int)sc.w[j], 0, (int)sc.x[i]);
        }
        lds_barrier();
    }
    if (a.S > 1)
        mx_store_part<TM, TN>(acc, a.part + (int64_t)blockIdx.z * a.M * a.ldp, a.ldp, m0 + wm, n0 + wn, a.M, a.N);
    else
        mx_store_tile<YT, TM, TN>(acc, smem + wave * mx_store_lds<YT, TM, TN>(), a.Y, a.ldy, m0 + wm, n0 + wn, a.M, a.N);
}

template <int YT, int TM, int TN>
static hipError_t launch_mx_gemm4_t(MxGemm4Args &a, hipStream_t s) {
    constexpr int BM = 64 * TM, BN = 64 * TN, lds = MxGemm4Lds<TM, TN>::template total<YT>();
    static_assert(lds <= 160 * 1024, "LDS budget");
    if (lds > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (hipError_t e = mx_allow_lds((const void *)mx_gemm4_kernel<YT, TM, TN>, lds, done)) return e;
    }
    a.tiles_m = (a.M + BM - 1) / BM;
    const dim3 grid((unsigned)(a.tiles_m * ((a.N + BN - 1) / BN)), 1, (unsigned)a.S);
    hipLaunchKernelGGL((mx_gemm4_kernel<YT, TM, TN>), grid, dim3(256), lds, s, a);
    return hipGetLastError();
}

template <int YT>
static hipError_t launch_mx_gemm4_y(MxGemm4Args &a, int kind, hipStream_t s) {
    return kind == MX_256x256 ? launch_mx_gemm4_t<YT, 4, 4>(a, s) : launch_mx_gemm4_t<YT, 2, 2>(a, s);
}

hipError_t launch_mx_gemm4(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s) {
    MxGemm4Args a = {(const uint8_t *)c.X, c.Xs, c.W, c.Ws, c.Y, c.ldy, (int)c.M, (int)(c.K / MX_BLOCK), (int)c.N};
    a.stages = (a.nb + 3) / 4;
    a.S = p.S;
    a.ldp = mx_ldp(c.N);
    a.part = p.S > 1 ? (float *)scratch : nullptr;
    const hipError_t e = c.x_dt == DT_F16 ? launch_mx_gemm4_y<DT_F16>(a, p.kind, s)
                       : c.x_dt == DT_BF16 ? launch_mx_gemm4_y<DT_BF16>(a, p.kind, s) : launch_mx_gemm4_y<DT_F32>(a, p.kind, s);
    return e == hipSuccess && p.S > 1 ? launch_mx_sum(a.part, p.S, c.Y, c.ldy, c.x_dt, c.M, c.N, s) : e;
}

}  // namespace mcq4
