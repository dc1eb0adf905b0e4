// Y[M, N] = X[M, K] W[N, K]^T with MXFP4 weights and 16-bit or fp32 X, through LDS, for many rows.
//
// A workgroup of four waves computes 32 TM rows x 128 TN columns, a wave all rows of its 32 TN
// columns, so that a weight is converted once per workgroup and feeds TM MFMAs
// (v_mfma_f32_32x32x16, the weights as the A operand: a lane ends up with four neighbouring
// columns of a row).
//
// A stage is 64 elements of K, two blocks.  Lane half h = l / 32 takes block h of its row and
// column for all four MFMAs of the stage: MFMA j multiplies dword j of the block's packed
// codes (8 elements) with X's elements 8 j .. 8 j + 7 of the same block.  So a lane needs 16
// bytes of codes and one scale a stage, and four v_cvt_scalef32_pk_*_fp4 make an operand.
//
// X goes through three stages of LDS, copied by all waves; a row's 16-byte chunk c lies at
// c ^ (row / 2) % 8, so that 16 lanes reading one chunk of 16 rows meet 16 banks.  A wave
// copies its own columns' codes two stages (64 bytes a column) at a time into a ring of three,
// chunk c at c ^ (column / 4) % 4, and their scales as the two aligned dwords that hold a
// column's four bytes.  Copies go out two stages ahead, between the MFMAs of a stage, as do
// the conversions and LDS reads of the next half stage; one barrier a stage.
//
// fp32 X (PIECES): three bf16 pieces that add up to it (mx_split_kernel), laid out as one row of
// 3 Kp elements, Kp = K rounded up to 128 with zeros; the weights are gone through three times.
//
// Few tiles: K is split over blockIdx.z, the partial sums added in order by mx_sum_kernel.
//
// Bound by the matrix cores and, on random operands, by power: 2048 x 4096 x 14336 fp16 takes
// 196 us (1.23 PFLOP/s) with the matrix cores 66% busy, where the library's product of plain
// fp16 matrices reaches 1.15 PFLOP/s on this card.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mx_gemm.h"

namespace mcq4 {

struct MxGemmArgs {
    const uint16_t *X;
    int64_t ldx;
    const uint8_t *W, *Ws;
    void *Y;
    int64_t ldy;
    int M, nb, N;          // nb: blocks of a weight row
    int kx;                // elements of a row of X (3 Kp with PIECES)
    int pairs, row_pairs;  // pairs of stages in all, and until the weights start anew
    int tiles_m, S;
    float *part;
    int64_t ldp;
    MxEpilogue epi;
};

template <int TM, int TN>
struct MxGemmLds {
    static constexpr int X_SLOT = 32 * TM * 128, W_SLOT = 32 * TN * 64, S_SLOT = 2 * 32 * TN * 4;
    static constexpr int W0 = 3 * X_SLOT, S0 = W0 + 4 * 3 * W_SLOT, LOOP = S0 + 4 * 3 * S_SLOT;
    template <int YT, bool EPI>
    static constexpr int total() { return std::max(LOOP, 4 * (EPI ? mx_epi_lds<TM, TN>() : mx_store_lds<YT, TM, TN>())); }
};

template <int XT, int YT, int TM, int TN, bool PIECES, bool EPI>
__global__ void __launch_bounds__(256, TM * TN >= 8 ? 1 : 2)
mx_gemm_kernel(MxGemmArgs a) {
    typedef MxGemmLds<TM, TN> L;
    constexpr int BM = 32 * TM, WN = 32 * TN, BN = 4 * WN;
    constexpr int NX = TM, NW = 2 * TN, NS = TN;               // copies of a wave: X per stage, codes and scales per pair
    constexpr int NMF = 2 * TM * TN;                           // MFMAs of a half stage
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lrow = lane & 31, lhi = lane >> 5;
    const MxTile tile = mx_tile(a.tiles_m);
    const int m0 = tile.m * BM, n0 = tile.n * BN;
    const int P0 = (int)((uint32_t)a.pairs * blockIdx.z / (uint32_t)a.S), P1 = (int)((uint32_t)a.pairs * (blockIdx.z + 1) / (uint32_t)a.S);
    const int np = P1 - P0;
    const int nk = PIECES ? 4 * np : min(4 * P1, a.nb) - 4 * P0;      // blocks
    const int nst = (nk + 1) >> 1, nfull = nk >> 1;

    const uint32_t lds0 = lds_addr(smem);
    uint8_t *const sX = smem, *const sW = smem + L::W0 + wave * 3 * L::W_SLOT, *const sS = smem + L::S0 + wave * 3 * L::S_SLOT;
    const uint32_t lW = lds0 + L::W0 + wave * 3 * L::W_SLOT, lS = lds0 + L::S0 + wave * 3 * L::S_SLOT;

    // Copies: the K position goes into the resource's base and size, so that nothing past an
    // array's end is read (it gives 0).
    const int x_row = (int)a.ldx * 2;
    const uint8_t *x_base = (const uint8_t *)(a.X + (int64_t)m0 * a.ldx + (int64_t)P0 * 128);
    const int x_bytes = (int)((int64_t)(min(a.M - m0, BM) - 1) * x_row + ((int64_t)a.kx - (int64_t)P0 * 128) * 2);
    const int vo_x0 = (8 * TM * wave + (lane >> 3)) * x_row + 16 * ((lane ^ (lane >> 4)) & 7);
    const int vo_x1 = (8 * TM * wave + (lane >> 3)) * x_row + 16 * ((lane ^ (4 + (lane >> 4))) & 7);
    const int w_row = a.nb * 16, rows_n = min(a.N - n0, BN);
    const uint8_t *w_base = a.W + (int64_t)n0 * w_row;
    const int w_bytes = rows_n * w_row;
    const int vo_w = (wave * WN + (lane >> 2)) * w_row + 16 * ((lane ^ (lane >> 4)) & 3);
    // Scales: from the aligned dword of the tile's first byte on; the last dword holds a byte of them.
    const uint8_t *s_first = a.Ws + (int64_t)n0 * a.nb;
    const int s_ph = (int)((uintptr_t)s_first & 3);
    const uint8_t *s_base = s_first - s_ph;
    const int s_bytes = (s_ph + rows_n * a.nb + 3) & ~3;
    const int vo_s = ((s_ph + (wave * WN + (TN == 2 ? lane : lrow)) * a.nb) & ~3) + (TN == 2 ? 0 : 4 * lhi);

    auto copy_x = [&](int s, int slot, int ci) {
        const int off = 128 * min(s, nst - 1);
        mx_copy16(mx_rsrc(x_base + off, x_bytes - off), sX + slot * L::X_SLOT + 128 * (8 * TM * wave + 8 * ci), ((ci & 1) ? vo_x1 : vo_x0) + 8 * ci * x_row, 0);
    };
    // Copy ci of pair p: NW of codes, then NS of scales.
    auto copy_w = [&](int p, int slot, int ci) {
        int pl = P0 + min(p, np - 1);
        if (PIECES) pl %= a.row_pairs;
        if (ci < NW) {
            const int off = 64 * pl;
            mx_copy16(mx_rsrc(w_base + off, w_bytes - off), sW + slot * L::W_SLOT + 1024 * ci, vo_w + 16 * ci * w_row, 0);
        } else {
            const int off = 4 * pl;
            mx_copy4(mx_rsrc(s_base + off, s_bytes - off), sS + slot * L::S_SLOT + 256 * (ci - NW), vo_s + 4 * (ci - NW), 0);
        }
    };

    // LDS reads.
    uint32_t x_off[4];                       // MFMA j: chunk 4 h + j of row l % 32
#pragma unroll
    for (int j = 0; j < 4; ++j) x_off[j] = lds0 + (uint32_t)(lrow * 128 + (((4 * lhi + j) ^ ((lrow >> 1) & 7)) << 4));
    auto read_x = [&](int slot, int j, int i) { return bitcast<half8_t>(mx_lds16(x_off[j] + slot * L::X_SLOT + i * 4096)); };
    uint32_t w_off[2], s_off[TN][2];         // stage parity
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        w_off[e] = lW + lrow * 64 + (((2 * e + lhi) ^ ((lrow >> 2) & 3)) << 4);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int p = ((s_ph + (wave * WN + 32 * j + lrow) * a.nb) & 3) + 2 * e + lhi;
            s_off[j][e] = lS + ((p >> 2) * WN + 32 * j + lrow) * 4 + (p & 3);
        }
    }
    struct Raw {
        uint4_t q[TN];
        float s[TN];
    };
    auto read_raw = [&](int pair, int slot, int e, int j, Raw &r) {
        r.q[j] = mx_lds16(w_off[e] + slot * L::W_SLOT + j * 2048);
        uint32_t b = *lds_ptr(s_off[j][e] + slot * L::S_SLOT);
        if (PIECES && 4 * ((P0 + pair) % a.row_pairs) + 2 * e + lhi >= a.nb) b = 0;       // X is 0 there
        r.s[j] = mx_scale(b);
    };
    auto convert = [&](uint32_t w, float s, int b) -> uint32_t {
        switch (b) {
            case 0: return mx_weights2<XT, 0>(w, s);
            case 1: return mx_weights2<XT, 1>(w, s);
            case 2: return mx_weights2<XT, 2>(w, s);
            default: return mx_weights2<XT, 3>(w, s);
        }
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // A half stage: the MFMAs of (Xc, Wc) and, between them, the conversion of the next half
    // stage's weights (dwords d0, d0 + 1 of raw), the read of its X (slot, from MFMA x_j on), the
    // raw weights of stage parity e of a pair where `reads`, and the copies given.
    auto half = [&](auto reads, auto n_copies, const half8_t (&Xc)[2][TM], half8_t (&Xn)[2][TM], const half8_t (&Wc)[2][TN], half8_t (&Wn)[2][TN],
                    const Raw &raw, int d0, int x_slot, int x_j, Raw &rn, int r_pair, int r_slot, int e, int s, int xs, int p, int ps) {
        constexpr int NC = decltype(n_copies)::value, CV = 8 * TN, XR = 2 * TM;
        uint4_t w[2][TN];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int idx = 0; idx < NMF; ++idx) {
            const int ks = idx / (TM * TN), i = (idx / TN) % TM, j = idx % TN;
            acc[i][j] = mfma32<XT>(Wc[ks][j], Xc[ks][i], acc[i][j]);
#pragma unroll
            for (int c = 0; c < CV; ++c)
                if (c * NMF / CV == idx) {
                    const int k = c / (4 * TN), jj = c / 4 % TN, b = c % 4;
                    w[k][jj][b] = convert(raw.q[jj][d0 + k], raw.s[jj], b);
                    if (b == 3) Wn[k][jj] = bitcast<half8_t>(w[k][jj]);
                }
            // X in the first half of the MFMAs, the raw weights behind it.
#pragma unroll
            for (int c = 0; c < XR; ++c)
                if (c * NMF / 2 / XR == idx) Xn[c / TM][c % TM] = read_x(x_slot, x_j + c / TM, c % TM);
            if constexpr (decltype(reads)::value)
#pragma unroll
                for (int c = 0; c < TN; ++c)
                    if (NMF / 2 + c == idx) read_raw(r_pair, r_slot, e, c, rn);
            if constexpr (NC > 0)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (c * NMF / NC == idx) {
                    if (c < NX) copy_x(s, xs, c);
                    else copy_w(p, ps, c - NX);
                }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int c = 0; c < NX; ++c) copy_x(s, s, c);
#pragma unroll
        for (int c = 0; c < NW + NS; ++c) copy_w(s, s, c);
    }
    wait_vmcnt<0>();
    lds_barrier();
    half8_t X0[2][TM], X1[2][TM], W0[2][TN], W1[2][TN];
    Raw R0, R1;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < TM; ++i) X0[k][i] = read_x(0, k, i);
#pragma unroll
    for (int j = 0; j < TN; ++j) read_raw(0, 0, 0, j, R0);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            uint4_t w;
#pragma unroll
            for (int b = 0; b < 4; ++b) w[b] = convert(R0.q[j][k], R0.s[j], b);
            W0[k][j] = bitcast<half8_t>(w);
        }

    // Stage s = 2 p + e: X in slot s % 3, the pair's weights in p % 3.  The barrier before a stage
    // makes the next one's X and weights visible (waited for by the wave that copied them) and
    // ends every wave's reads of the stage before, whose slots this stage's copies fill: X of
    // stage s + 2 in every stage, codes and scales of pair p + 2 in an odd one.  vmcnt is in
    // order: an odd stage leaves its pair's copies behind X's in flight.
    typedef std::integral_constant<int, 0> none;
    int x0 = 0, x1 = 1, x2 = 2, w0 = 0, w1 = 1, w2 = 2;
    auto stage = [&](auto odd, int s, Raw &rc, Raw &rn) {
        constexpr bool ODD = decltype(odd)::value;
        if (s > 0) {
            if constexpr (ODD) wait_vmcnt<0>();
            else wait_vmcnt<NW + NS>();
            lds_barrier();
        }
        const int p = s >> 1;
        half(std::true_type{}, std::integral_constant<int, ODD ? NX + NW + NS : NX>{}, X0, X1, W0, W1, rc, 2, x0, 2,
             rn, ODD ? p + 1 : p, ODD ? w1 : w0, ODD ? 0 : 1, s + 2, x2, p + 2, w2);
        half(std::false_type{}, none{}, X1, X0, W1, W0, rn, 0, x1, 0, rn, 0, 0, 0, 0, 0, 0, 0);
        const int t = x0;
        x0 = x1; x1 = x2; x2 = t;
        if (ODD) {
            const int u = w0;
            w0 = w1; w1 = w2; w2 = u;
        }
    };
    int s = 0;
    for (; s + 1 < nfull; s += 2) {
        stage(std::false_type{}, s, R0, R1);
        stage(std::true_type{}, s + 1, R1, R0);
    }
    if (s < nfull) stage(std::false_type{}, s, R0, R1);
    wait_vmcnt<0>();
    lds_barrier();
    if (nk & 1) {
        // One block left: both lane halves take it, half h the dword 2 j + h in MFMA j.
        const int st = nfull, e = st & 1;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            half8_t w[TN];
#pragma unroll
            for (int jj = 0; jj < TN; ++jj) {
                const int p = ((s_ph + (wave * WN + 32 * jj + lrow) * a.nb) & 3) + 2 * e;
                const uint4_t q = mx_lds16(lW + w0 * L::W_SLOT + jj * 2048 + lrow * 64 + (((2 * e) ^ ((lrow >> 2) & 3)) << 4));
                const float sc = mx_scale(*lds_ptr(lS + w0 * L::S_SLOT + ((p >> 2) * WN + 32 * jj + lrow) * 4 + (p & 3)));
                w[jj] = bitcast<half8_t>(mx_weights8<XT>(lhi ? q[2 * j + 1] : q[2 * j], sc));
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const half8_t x = bitcast<half8_t>(mx_lds16(lds0 + x0 * L::X_SLOT + i * 4096 + lrow * 128 + (((2 * j + lhi) ^ ((lrow >> 1) & 7)) << 4)));
#pragma unroll
                for (int jj = 0; jj < TN; ++jj) acc[i][jj] = mfma32<XT>(w[jj], x, acc[i][jj]);
            }
        }
        lds_barrier();
    }
    if (a.S > 1)
        mx_store_part<TM, TN>(acc, a.part + (int64_t)blockIdx.z * a.M * a.ldp, a.ldp, m0, n0 + wave * WN, a.M, a.N);
    else if constexpr (EPI)
        mx_store_epi<YT, TM, TN>(acc, smem + wave * mx_epi_lds<TM, TN>(), a.epi, a.Y, a.ldy, m0, n0 + wave * WN, a.M, a.N);
    else
        mx_store_tile<YT, TM, TN>(acc, smem + wave * mx_store_lds<YT, TM, TN>(), a.Y, a.ldy, m0, n0 + wave * WN, a.M, a.N);
}

// fp32 rows to three bf16 pieces, [M][3][Kp].  Each piece is the upper half of what the ones
// before it left (cut off, not rounded: the largest finite values stay finite), so the three
// hold all 24 bits; an infinity or NaN is its first piece alone.
__global__ void __launch_bounds__(256)
mx_split_kernel(const float *__restrict__ X, int64_t ldx, int M, int K, int Kp, uint16_t *__restrict__ out) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int k8 = Kp >> 3;
    if (u >= (int64_t)M * k8) return;
    const int m = (int)(u / k8), k = (int)(u % k8) * 8;
    uint4_t p[3] = {};
    if (k < K) {
        const float4_t *x = (const float4_t *)(X + (int64_t)m * ldx + k);
        const float4_t v0 = x[0], v1 = x[1];
        const float f[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        mx_split8(f, p);
    }
#pragma unroll
    for (int s = 0; s < 3; ++s) *(uint4_t *)(out + ((int64_t)m * 3 + s) * Kp + k) = p[s];
}

hipError_t launch_mx_split(const MxCall &c, uint16_t *out, hipStream_t s) {
    const int Kp = (int)((c.K + 127) / 128 * 128);
    const int64_t units = c.M * (Kp / 8);
    hipLaunchKernelGGL(mx_split_kernel, dim3((unsigned)((units + 255) / 256)), dim3(256), 0, s, (const float *)c.X, c.ldx, (int)c.M, (int)c.K, Kp, out);
    return hipGetLastError();
}

template <int DT, bool EPI>
__global__ void __launch_bounds__(256)
mx_sum_kernel(const float *__restrict__ part, int S, void *Y, int64_t ldy, int M, int N, int64_t ldp, bool vec, MxEpilogue epi) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t n4 = ldp >> 2;
    if (u >= M * n4) return;
    const int m = (int)(u / n4), n = (int)(u % n4) * 4;
    const float4_t *p = (const float4_t *)part + u;
    MxOperands<DT, 4> ops;
    if constexpr (EPI) ops.load(epi, m, n, M, N);
    float4_t v = p[0];
    for (int s = 1; s < S; ++s) v += p[(int64_t)s * M * n4];
    if constexpr (EPI) {
        float f[4] = {v[0], v[1], v[2], v[3]};
        mx_finish<DT, 4>(epi, ops, f);
        v = float4_t{f[0], f[1], f[2], f[3]};
    }
    const int64_t o = (int64_t)m * ldy + n;
    if (vec && n + 4 <= N) {
        if constexpr (DT == DT_F32) *(float4_t *)((float *)Y + o) = v;
        else *(uint2_t *)((uint16_t *)Y + o) = uint2_t{mx_pair<DT>(v[0], v[1]), mx_pair<DT>(v[2], v[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < N) mx_store<DT>(Y, o + e, v[e]);
    }
}

template <bool EPI>
static hipError_t launch_mx_sum_t(const float *part, int S, void *Y, int64_t ldy, int dt, int64_t M, int64_t N, const MxEpilogue &epi, hipStream_t s) {
    const int64_t ldp = mx_ldp(N);
    const dim3 grid((unsigned)((M * (ldp >> 2) + 255) / 256)), block(256);
    const bool vec = (ldy & 3) == 0 && (uintptr_t)Y % 16 == 0;
    if (dt == DT_F16) hipLaunchKernelGGL((mx_sum_kernel<DT_F16, EPI>), grid, block, 0, s, part, S, Y, ldy, (int)M, (int)N, ldp, vec, epi);
    else if (dt == DT_BF16) hipLaunchKernelGGL((mx_sum_kernel<DT_BF16, EPI>), grid, block, 0, s, part, S, Y, ldy, (int)M, (int)N, ldp, vec, epi);
    else hipLaunchKernelGGL((mx_sum_kernel<DT_F32, EPI>), grid, block, 0, s, part, S, Y, ldy, (int)M, (int)N, ldp, vec, epi);
    return hipGetLastError();
}
hipError_t launch_mx_sum(const float *part, int S, void *Y, int64_t ldy, int dt, int64_t M, int64_t N, const MxEpilogue *epi, hipStream_t s) {
    return epi ? launch_mx_sum_t<true>(part, S, Y, ldy, dt, M, N, *epi, s) : launch_mx_sum_t<false>(part, S, Y, ldy, dt, M, N, MxEpilogue{}, s);
}

template <int XT, int YT, int TM, int TN, bool PIECES, bool EPI>
static hipError_t launch_mx_gemm_t(MxGemmArgs &a, hipStream_t s) {
    constexpr int BM = 32 * TM, BN = 128 * TN, lds = MxGemmLds<TM, TN>::template total<YT, EPI>();
    static_assert(lds <= 160 * 1024, "LDS budget");
    if (lds > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (hipError_t e = mx_allow_lds((const void *)mx_gemm_kernel<XT, YT, TM, TN, PIECES, EPI>, lds, done)) return e;
    }
    a.tiles_m = (a.M + BM - 1) / BM;
    const dim3 grid((unsigned)(a.tiles_m * ((a.N + BN - 1) / BN)), 1, (unsigned)a.S);
    hipLaunchKernelGGL((mx_gemm_kernel<XT, YT, TM, TN, PIECES, EPI>), grid, dim3(256), lds, s, a);
    return hipGetLastError();
}

template <int XT, int YT, bool PIECES, bool EPI>
static hipError_t launch_mx_gemm_e(MxGemmArgs &a, int kind, hipStream_t s) {
    return kind == 1 ? launch_mx_gemm_t<XT, YT, 8, 2, PIECES, EPI>(a, s)
         : kind == 2 ? launch_mx_gemm_t<XT, YT, 4, 2, PIECES, EPI>(a, s)
         : kind == 3 ? launch_mx_gemm_t<XT, YT, 4, 1, PIECES, EPI>(a, s) : launch_mx_gemm_t<XT, YT, 2, 1, PIECES, EPI>(a, s);
}
// With K split the epilogue is mx_sum_kernel's.
template <int XT, int YT, bool PIECES>
static hipError_t launch_mx_gemm_x(MxGemmArgs &a, int kind, const MxEpilogue *epi, hipStream_t s) {
    if (!epi || a.S > 1) return launch_mx_gemm_e<XT, YT, PIECES, false>(a, kind, s);
    a.epi = *epi;
    return launch_mx_gemm_e<XT, YT, PIECES, true>(a, kind, s);
}

hipError_t launch_mx_gemm(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s) {
    MxGemmArgs a = {(const uint16_t *)c.X, c.ldx, c.W, c.Ws, c.Y, c.ldy, (int)c.M, (int)(c.K / MX_BLOCK), (int)c.N, (int)c.K};
    a.row_pairs = a.pairs = (a.nb + 3) / 4;
    a.S = p.S;
    a.ldp = mx_ldp(c.N);
    a.part = p.S > 1 ? (float *)scratch : nullptr;
    hipError_t e;
    if (c.x_dt == DT_F32) {
        const int Kp = 128 * a.row_pairs;
        uint16_t *pieces = (uint16_t *)scratch;
        if ((e = launch_mx_split(c, pieces, s)) != hipSuccess) return e;
        a.X = pieces;
        a.kx = 3 * Kp;
        a.ldx = a.kx;
        a.pairs = 3 * a.row_pairs;
        if (p.S > 1) a.part = (float *)(pieces + mx_pieces(c.M, c.K));
        e = launch_mx_gemm_x<DT_BF16, DT_F32, true>(a, p.kind, c.epi, s);
    } else {
        e = c.x_dt == DT_BF16 ? launch_mx_gemm_x<DT_BF16, DT_BF16, false>(a, p.kind, c.epi, s) : launch_mx_gemm_x<DT_F16, DT_F16, false>(a, p.kind, c.epi, s);
    }
    if (e == hipSuccess && p.S > 1) e = launch_mx_sum(a.part, p.S, c.Y, c.ldy, c.x_dt, c.M, c.N, c.epi, s);
    return e;
}

}  // namespace mcq4
