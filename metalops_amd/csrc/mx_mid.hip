// MXFP4 products of a few dozen to a few hundred rows: K is split over a workgroup's waves.
//
// With few output tiles a kernel that shares stages of K between waves spends its time at the
// barriers, waiting for copies that it sent out a stage ahead.  Here each wave (of four, or of
// eight with 32 rows) has a range of K of its own and computes the whole tile of 32 TM rows x
// 32 TN columns over it, from its own ring of NS stages in LDS: no barrier before the waves'
// sums are added (in wave order), and as many independent streams of copies in flight.  Nothing
// is read twice by a workgroup, since the waves' parts of X and W are different ones.
// 16 x 14336 x 4096, bf16: 20.6 us with the direct kernel, 11.5 here; the weights alone take 6.4
// at the rate of a large copy, and the rest is the start, the ring's first loads and the joins.
//
// Operands, LDS swizzles and the conversion of weights are those of mx_gemm.hip (16-bit or
// fp32 X; a stage is 64 elements of K) and mx_gemm4.hip (microscaled X; 128 elements).
//
// Where that still leaves most CUs without work, blockIdx.z splits K further.  A workgroup then
// writes its sums through to memory (agent scope: the XCDs' L2s are not coherent), draws a
// ticket, and the last one of a tile adds all of them in the order of K.
#include <algorithm>
#include <type_traits>

#include "mx_gemm.h"

namespace mcq4 {

struct MxMidArgs {
    const uint8_t *X, *Xs;
    int64_t ldx;           // bytes
    const uint8_t *W, *Ws;
    void *Y;
    int64_t ldy;
    int M, nb, N;
    int kx;                // bytes of a row of X
    int units, row_units;  // 128 elements of K each, in all and until the weights start anew
    int tiles_m, S;
    float *part;
    uint32_t *tickets;
    MxEpilogue epi;
};

__device__ __forceinline__ void mx_wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xC07F);          // lgkmcnt(0)
    asm volatile("" ::: "memory");
}
template <int N>
__device__ __forceinline__ void mx_wait_copies() {
    wait_vmcnt<N>();
    asm volatile("" ::: "memory");
}

// The waves' tiles added in LDS, then over the splits, and stored.
template <int YT, int TM, int TN, int WAVES, bool EPI>
__device__ __forceinline__ void mx_join(const float16_t (&acc)[TM][TN], float *lds, const MxMidArgs &a, MxTile tile) {
    constexpr int BM = 32 * TM, BN = 32 * TN, PITCH = BN + 4, U = BM * BN / 4, THREADS = 64 * WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 31, hi = lane >> 5;
    const int m0 = tile.m * BM, n0 = tile.n * BN;
    constexpr int EACH = (U + THREADS - 1) / THREADS;
    MxOperands<YT, 4> ops[EACH];
    auto operands = [&](int i) {
        const int u = tid + i * THREADS;
        if (u < U) ops[i].load(a.epi, m0 + u / (BN / 4), n0 + 4 * (u % (BN / 4)), a.M, a.N);
    };
    if constexpr (EPI)
        if (a.S == 1)
#pragma unroll
            for (int i = 0; i < EACH; ++i) operands(i);
    __syncthreads();                              // every wave is done with its ring
    float *mine = lds + wave * BM * PITCH;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(float4_t *)(mine + (32 * i + row) * PITCH + 32 * j + 8 * q + 4 * hi) =
                    float4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __syncthreads();
    auto sum = [&](int u) {
        const float *p = lds + (u / (BN / 4)) * PITCH + 4 * (u % (BN / 4));
        float4_t v = *(const float4_t *)p;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += *(const float4_t *)(p + w * BM * PITCH);
        return v;
    };
    const bool vec = (a.ldy & 3) == 0 && ((uintptr_t)a.Y & 15) == 0;
    auto store = [&](int i, int u, float4_t v) {
        const int m = m0 + u / (BN / 4), n = n0 + 4 * (u % (BN / 4));
        if (m >= a.M || n >= a.N) return;
        const int64_t o = (int64_t)m * a.ldy + n;
        if constexpr (EPI) {
            float f[4] = {v[0], v[1], v[2], v[3]};
            mx_finish<YT, 4>(a.epi, ops[i], f);
            v = float4_t{f[0], f[1], f[2], f[3]};
        }
        if (vec && n + 4 <= a.N) {
            if constexpr (YT == DT_F32) *(float4_t *)((float *)a.Y + o) = v;
            else *(uint2_t *)((uint16_t *)a.Y + o) = uint2_t{mx_pair<YT>(v[0], v[1]), mx_pair<YT>(v[2], v[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < a.N) mx_store<YT>(a.Y, o + e, v[e]);
        }
    };
    if (a.S == 1) {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (tid + i * THREADS < U) store(i, tid + i * THREADS, sum(tid + i * THREADS));
        return;
    }
    constexpr int SC1 = 16;                       // agent scope: past the XCD's L2
    const int t = tile.n * a.tiles_m + tile.m;
    const __amdgpu_buffer_rsrc_t rs = mx_rsrc(a.part + (int64_t)t * a.S * (BM * BN), (int64_t)a.S * (BM * BN * 4));
#pragma unroll
    for (int u = tid; u < U; u += THREADS)
        __builtin_amdgcn_raw_buffer_store_b128(bitcast<uint4_t>(sum(u)), rs, 16 * u, (int)blockIdx.z * (BM * BN * 4), SC1);
    __builtin_amdgcn_s_waitcnt(0x0F70);           // vmcnt(0): the sums are in memory
    __syncthreads();
    int *last = (int *)lds;
    if (tid == 0) {
        const uint32_t before = __hip_atomic_fetch_add(&a.tickets[t], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = before == (uint32_t)a.S - 1;
        if (*last) __hip_atomic_store(&a.tickets[t], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    if constexpr (EPI)
#pragma unroll
        for (int i = 0; i < EACH; ++i) operands(i);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int u = tid + i * THREADS;
        if (u >= U) break;
        float4_t v = bitcast<float4_t>(__builtin_amdgcn_raw_buffer_load_b128(rs, 16 * u, 0, SC1));
        for (int z = 1; z < a.S; ++z) v += bitcast<float4_t>(__builtin_amdgcn_raw_buffer_load_b128(rs, 16 * u, z * (BM * BN * 4), SC1));
        store(i, u, v);
    }
}
template <int TM, int TN, int WAVES>
constexpr int mx_join_lds() { return WAVES * 32 * TM * (32 * TN + 4) * 4; }

// ---- 16-bit X, or three bf16 pieces of fp32 X -------------------------------------------------

// XR: rows of X in LDS, fewer than 32 TM where a call has no more; the MFMA's other rows repeat them.
template <int TM, int TN, int NS, int XR, int WAVES>
struct MxMidLds {
    static constexpr int NP = NS / 2 + 1;                        // pairs of stages whose codes and scales are held
    static constexpr int X_SLOT = XR * 128, W_SLOT = 32 * TN * 64, S_SLOT = 2 * 32 * TN * 4;
    static constexpr int W0 = NS * X_SLOT, S0 = W0 + NP * W_SLOT, WAVE = S0 + NP * S_SLOT;
    static constexpr int TOTAL = std::max(WAVES * WAVE, mx_join_lds<TM, TN, WAVES>()), WGS = TOTAL > 80 * 1024 ? 1 : 2;
};

template <int XT, int YT, int TM, int TN, int NS, int XR, int WAVES, bool PIECES, bool EPI>
__global__ void __launch_bounds__(64 * WAVES, (MxMidLds<TM, TN, NS, XR, WAVES>::WGS))
mx_mid_kernel(MxMidArgs a) {
    typedef MxMidLds<TM, TN, NS, XR, WAVES> L;
    static_assert(XR == 32 * TM || (TM == 1 && XR < 32), "rows of X");
    
    constexpr int BM = 32 * TM, BN = 32 * TN;
    // Copies of every stage (X), and of an even one besides: the pair's scales and its codes, 64 bytes a column.
    constexpr int EVERY = XR / 8, NSC = TN, EVEN = NSC + 2 * TN;
    static_assert((NS - 1) * EVERY + (NS - 1) / 2 * EVEN < 64, "vmcnt");
    constexpr int NMF = 2 * TM * TN;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lrow = lane & 31, lhi = lane >> 5;
    const MxTile tile = mx_tile(a.tiles_m);
    const int m0 = tile.m * BM, n0 = tile.n * BN;
    const uint32_t part = blockIdx.z * WAVES + wave, parts = a.S * WAVES;
    const int P0 = (int)((uint32_t)a.units * part / parts), P1 = (int)((uint32_t)a.units * (part + 1) / parts);
    const int nk = max(0, PIECES ? 4 * (P1 - P0) : min(4 * P1, a.nb) - 4 * P0);      // blocks
    const int nst = (nk + 1) >> 1, nfull = nk >> 1;

    uint8_t *const ring = smem + wave * L::WAVE;
    const uint32_t lds0 = lds_addr(ring);
    const int x_row = (int)a.ldx, w_row = a.nb * 16;
    const int rows_m = min(a.M - m0, XR), rows_n = min(a.N - n0, BN);
    const uint8_t *x_base = a.X + (int64_t)m0 * a.ldx + (int64_t)P0 * 256;
    const int x_bytes = (rows_m - 1) * x_row + a.kx - P0 * 256;
    const uint8_t *w_base = a.W + (int64_t)n0 * w_row;
    const int w_bytes = rows_n * w_row;
    const int vo_x0 = (lane >> 3) * x_row + 16 * ((lane ^ (lane >> 4)) & 7);
    const int vo_x1 = (lane >> 3) * x_row + 16 * ((lane ^ (4 + (lane >> 4))) & 7);
    const int vo_w = (lane >> 2) * w_row + 16 * ((lane ^ (lane >> 4)) & 3);           // chunk c of a column at c ^ (column / 4) % 4
    const uint8_t *s_first = a.Ws + (int64_t)n0 * a.nb;
    const int s_ph = (int)((uintptr_t)s_first & 3);
    const int s_bytes = (s_ph + rows_n * a.nb + 3) & ~3;

    // Past this wave's range a copy brings zeros and reads nothing: every stage sends out as many.
    auto copy_x = [&](int s, int slot, int c) {
        const int off = 128 * s;
        mx_copy16(mx_rsrc(x_base + off, s < nst ? x_bytes - off : 0), ring + slot * L::X_SLOT + 1024 * c, ((c & 1) ? vo_x1 : vo_x0) + 8 * c * x_row, 0);
    };
    // Copy c of pair p: its scales, then its codes.
    auto copy_even = [&](int p, int slot, int c) {
        int pl = P0 + p;
        if (PIECES) pl %= a.row_units;
        if (c >= NSC) {
            const int off = 64 * pl;
            mx_copy16(mx_rsrc(w_base + off, 2 * p < nst ? w_bytes - off : 0), ring + L::W0 + slot * L::W_SLOT + 1024 * (c - NSC), vo_w + 16 * (c - NSC) * w_row, 0);
            return;
        }
        const int off = 4 * pl, e = 64 * c + lane, col = e % BN, d = e / BN;
        mx_copy4(mx_rsrc(s_first - s_ph + off, 2 * p < nst ? s_bytes - off : 0), ring + L::S0 + slot * L::S_SLOT + 256 * c, ((s_ph + col * a.nb) & ~3) + 4 * d, 0);
    };

    uint32_t x_off[4];
    const int xrow = lrow & (XR - 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) x_off[j] = lds0 + (uint32_t)(xrow * 128 + (((4 * lhi + j) ^ ((xrow >> 1) & 7)) << 4));
    auto read_x = [&](int slot, int j, int i) { return bitcast<half8_t>(mx_lds16(x_off[j] + slot * L::X_SLOT + i * 4096)); };
    uint32_t w_off[2];                           // stage parity
#pragma unroll
    for (int e = 0; e < 2; ++e)
        w_off[e] = lds0 + L::W0 + lrow * 64 + (((2 * e + lhi) ^ ((lrow >> 2) & 3)) << 4);
    uint32_t s_off[TN][2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int p = ((s_ph + (32 * j + lrow) * a.nb) & 3) + 2 * e + lhi;
            s_off[j][e] = lds0 + L::S0 + ((p >> 2) * BN + 32 * j + lrow) * 4 + (p & 3);
        }
    struct Raw {
        uint4_t q[TN];
        uint32_t s[TN];                          // the scale's byte
    };
    auto read_raw = [&](int s, int pslot, int e, int j, Raw &r) {
        r.q[j] = mx_lds16(w_off[e] + pslot * L::W_SLOT + j * 2048);
        uint32_t b = *lds_ptr(s_off[j][e] + pslot * L::S_SLOT);
        if (PIECES && 4 * ((P0 + (s >> 1)) % a.row_units) + 2 * e + lhi >= a.nb) b = 0;          // X is 0 there
        r.s[j] = b;
    };
    auto convert = [&](uint32_t w, uint32_t byte, int b) -> uint32_t {
        const float s = mx_scale(byte);
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

    // A half stage, as in mx_gemm.hip.  SECOND: it reads the next stage's X and sends out copies
    // into the slot of this one; else it reads this stage's X and the next stage's weights.
    auto half = [&](auto second, auto odd, int s, int slot, int nslot, int pslot, const half8_t (&Xc)[2][TM], half8_t (&Xn)[2][TM],
                    const half8_t (&Wc)[2][TN], half8_t (&Wn)[2][TN], const Raw &raw, Raw &rn) {
        constexpr bool SECOND = decltype(second)::value, ODD = decltype(odd)::value;
        constexpr int CV = 8 * TN, RD = 2 * TM;
        // Stage s + NS is even: what comes by pairs goes first.
        constexpr int SC = SECOND && ((NS + (ODD ? 1 : 0)) % 2 == 0) ? EVEN : 0, NC = SECOND ? SC + EVERY : 0;
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
                    w[k][jj][b] = convert(raw.q[jj][(SECOND ? 0 : 2) + k], raw.s[jj], b);
                    if (b == 3) Wn[k][jj] = bitcast<half8_t>(w[k][jj]);
                }
#pragma unroll
            for (int c = 0; c < RD; ++c)
                if (c * NMF / 2 / RD == idx) Xn[c / TM][c % TM] = read_x(SECOND ? nslot : slot, (SECOND ? 0 : 2) + c / TM, c % TM);
            if constexpr (!SECOND)
#pragma unroll
                for (int c = 0; c < TN; ++c)
                    if (NMF / 2 + c * NMF / 2 / TN == idx) read_raw(s + 1, pslot, ODD ? 0 : 1, c, rn);
            if constexpr (NC > 0)
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    if (c * NMF / NC == idx) {
                        if (c < SC) copy_even((s + NS) >> 1, pslot, c);
                        else copy_x(s + NS, slot, c - SC);
                    }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (nk > 0) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if ((s & 1) == 0)
#pragma unroll
                for (int c = 0; c < EVEN; ++c) copy_even(s >> 1, (s >> 1) % L::NP, c);
#pragma unroll
            for (int c = 0; c < EVERY; ++c) copy_x(s, s, c);
        }
        mx_wait_copies<(NS - 1) * EVERY + (NS - 1) / 2 * EVEN>();
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
        // Stage s lies in slot s % NS, what comes by pairs in slot (s / 2) % NP.  Stage s + 1 has to be there
        // before stage s starts: all but the copies of the newest NS - 2 stages, s + 2 the first of them.
        int slot = 0, pslot = 0;
        auto next = [](int v, int n) { return v + 1 == n ? 0 : v + 1; };
        auto stage = [&](auto odd, int s, Raw &rc, Raw &rn) {
            constexpr bool ODD = decltype(odd)::value;
            const int nslot = next(slot, NS);
            const int np = ODD ? next(pslot, L::NP) : pslot;                   // pair of stage s + 1
            // Pair (s + NS) / 2, where that is even, counted from this stage's pair.
            constexpr int AHEAD = (NS + (ODD ? 1 : 0)) / 2;
            int cp = pslot;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) cp = next(cp, L::NP);
            mx_wait_copies<(NS - 2) * EVERY + (ODD ? (NS - 2) / 2 : (NS - 1) / 2) * EVEN>();
            half(std::false_type{}, odd, s, slot, nslot, np, X0, X1, W0, W1, rc, rn);
            mx_wait_lds();                                                     // this stage's slot has been read
            half(std::true_type{}, odd, s, slot, nslot, cp, X1, X0, W1, W0, rn, rn);
            slot = nslot;
            pslot = np;
        };
        int s = 0;
        for (; s + 1 < nfull; s += 2) {
            stage(std::false_type{}, s, R0, R1);
            stage(std::true_type{}, s + 1, R1, R0);
        }
        if (s < nfull) stage(std::false_type{}, s, R0, R1);
        mx_wait_copies<0>();
        if (nk & 1) {
            // One block left: both lane halves take it, half h the dword 2 j + h in MFMA j.
            const int e = nfull & 1;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                half8_t w[TN];
#pragma unroll
                for (int jj = 0; jj < TN; ++jj) {
                    const int p = ((s_ph + (32 * jj + lrow) * a.nb) & 3) + 2 * e;
                    const uint4_t q = mx_lds16(lds0 + L::W0 + pslot * L::W_SLOT + jj * 2048 + lrow * 64 + (((2 * e) ^ ((lrow >> 2) & 3)) << 4));
                    const float sc = mx_scale(*lds_ptr(lds0 + L::S0 + pslot * L::S_SLOT + ((p >> 2) * BN + 32 * jj + lrow) * 4 + (p & 3)));
                    w[jj] = bitcast<half8_t>(mx_weights8<XT>(lhi ? q[2 * j + 1] : q[2 * j], sc));
                }
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const half8_t x = bitcast<half8_t>(mx_lds16(lds0 + slot * L::X_SLOT + i * 4096 + xrow * 128 + (((2 * j + lhi) ^ ((xrow >> 1) & 7)) << 4)));
#pragma unroll
                    for (int jj = 0; jj < TN; ++jj) acc[i][jj] = mfma32<XT>(w[jj], x, acc[i][jj]);
                }
            }
        }
    }
    mx_join<YT, TM, TN, WAVES, EPI>(acc, (float *)smem, a, tile);
}

// ---- microscaled X ---------------------------------------------------------------------------

template <int TM, int TN, int NS, int WAVES>
struct MxMid4Lds {
    static constexpr int ROWS = 32 * (TM + TN), SLOT = ROWS * 64;                          // X's rows, then W's
    static constexpr int SX = (TM + 1) / 2 * 64, SR = SX + (TN + 1) / 2 * 64, S_SLOT = SR * 16;   // rows of scales
    static constexpr int NG = NS / 4 + 2;                        // pieces of 16 scales that are held
    static constexpr int S0 = NS * SLOT, WAVE = S0 + NG * S_SLOT;
    static constexpr int TOTAL = std::max(WAVES * WAVE, mx_join_lds<TM, TN, WAVES>()), WGS = TOTAL > 80 * 1024 ? 1 : 2;
};

template <int YT, int TM, int TN, int NS, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, (MxMid4Lds<TM, TN, NS, WAVES>::WGS))
mx_mid4_kernel(MxMidArgs a) {
    typedef MxMid4Lds<TM, TN, NS, WAVES> L;
    constexpr int BM = 32 * TM, BN = 32 * TN;
    constexpr int NX = 2 * TM, G = 2 * (TM + TN), NSC = L::SR / 64;
    constexpr int NMF = TM * TN;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lrow = lane & 31, lhi = lane >> 5;
    const MxTile tile = mx_tile(a.tiles_m);
    const int m0 = tile.m * BM, n0 = tile.n * BN;
    const uint32_t part = blockIdx.z * WAVES + wave, parts = a.S * WAVES;
    const int s0 = (int)((uint32_t)a.units * part / parts), s1 = (int)((uint32_t)a.units * (part + 1) / parts);
    const int nk = max(0, min(4 * s1, a.nb) - 4 * s0), nst = s1 - s0, nfull = nk >> 2;

    uint8_t *const ring = smem + wave * L::WAVE;
    const uint32_t lds0 = lds_addr(ring);
    const int row = a.nb * 16;
    const int rows_m = min(a.M - m0, BM), rows_n = min(a.N - n0, BN);
    const uint8_t *x_base = a.X + (int64_t)m0 * row + (int64_t)s0 * 64, *w_base = a.W + (int64_t)n0 * row + (int64_t)s0 * 64;
    const int x_bytes = rows_m * row - s0 * 64, w_bytes = rows_n * row - s0 * 64;
    const int vo_c = (lane >> 2) * row + 16 * ((lane ^ (lane >> 4)) & 3);
    auto copy = [&](int s, int slot, int c) {
        const int off = 64 * s, r = 16 * (c < NX ? c : c - NX);
        const uint8_t *base = c < NX ? x_base : w_base;
        mx_copy16(mx_rsrc(base + off, s < nst ? (c < NX ? x_bytes : w_bytes) - off : 0), ring + slot * L::SLOT + 1024 * c, vo_c + r * row, 0);
    };
    const uint8_t *xs_first = a.Xs + (int64_t)m0 * a.nb + 4 * s0, *ws_first = a.Ws + (int64_t)n0 * a.nb + 4 * s0;
    const int x_ph = (int)((uintptr_t)xs_first & 3), w_ph = (int)((uintptr_t)ws_first & 3);
    const int xs_bytes = (x_ph + rows_m * a.nb - 4 * s0 + 3) & ~3, ws_bytes = (w_ph + rows_n * a.nb - 4 * s0 + 3) & ~3;
    // Piece g of every row's scales: its aligned dwords 4 g .. 4 g + 3; 64 rows a copy, X's and W's
    // from a multiple of 64 on (with an odd TM or TN also rows of the next tile, or none).
    auto copy_s = [&](int g, int slot, int c) {
        const int off = 16 * g, r = 64 * c + lane;
        const bool is_x = 64 * c < L::SX;
        mx_copy16(mx_rsrc((is_x ? xs_first - x_ph : ws_first - w_ph) + off, 4 * g <= nst ? (is_x ? xs_bytes : ws_bytes) - off : 0),
                  ring + L::S0 + slot * L::S_SLOT + 1024 * c, (is_x ? x_ph + r * a.nb : w_ph + (r - L::SX) * a.nb) & ~3, 0);
    };

    uint32_t d_off[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) d_off[t] = lds0 + lrow * 64 + (((2 * lhi + t) ^ ((lrow >> 2) & 3)) << 4);
    auto read_x = [&](int slot, int t, int i) { return mx_lds16(d_off[t] + slot * L::SLOT + i * 2048); };
    auto read_w = [&](int slot, int t, int j) { return mx_lds16(d_off[t] + slot * L::SLOT + (TM + j) * 2048); };
    auto read_s = [&](int d, int r) { return mx_lds4(lds0 + L::S0 + (int)((uint32_t)(d >> 2) % L::NG) * L::S_SLOT + (r + lrow) * 16 + 4 * (d & 3)); };
    uint32_t sh_x[TM], sh_w[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) sh_x[i] = 8 * (((x_ph + (32 * i + lrow) * a.nb) & 3) + 2 * lhi);
#pragma unroll
    for (int j = 0; j < TN; ++j) sh_w[j] = 8 * (((w_ph + (32 * j + lrow) * a.nb) & 3) + 2 * lhi);
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
    if (nk > 0) {
        Step A, B;
        Scales now, lo, hi;
#pragma unroll
        for (int g = 0; g < (NS + 3) / 4 + 1; ++g)
#pragma unroll
            for (int c = 0; c < NSC; ++c) copy_s(g, g, c);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int c = 0; c < G; ++c) copy(s, s, c);
        mx_wait_copies<(NS - 1) * G>();
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            A.x[i] = read_x(0, 0, i);
            lo.x[i] = read_s(1, 32 * i);
            now.x[i] = pick(read_s(0, 32 * i), lo.x[i], sh_x[i]);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            A.w[j] = read_w(0, 0, j);
            lo.w[j] = read_s(1, L::SX + 32 * j);
            now.w[j] = pick(read_s(0, L::SX + 32 * j), lo.w[j], sh_w[j]);
        }
        int slot = 0;
        for (int s = 0; s < nfull; ++s) {
            const int nslot = slot + 1 == NS ? 0 : slot + 1;
            mx_wait_copies<(NS - 2) * G>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int idx = 0; idx < NMF; ++idx) {
                const int i = idx / TN, j = idx % TN;
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(A.w[j]), mx_operand(A.x[i]), acc[i][j], 4, 4,
                                                                            0, (int)now.w[j], 0, (int)now.x[i]);
#pragma unroll
                for (int c = 0; c < TM + TN; ++c) {
                    if (c * NMF / (TM + TN) == idx) {
                        if (c < TM) B.x[c] = read_x(slot, 1, c);
                        else B.w[c - TM] = read_w(slot, 1, c - TM);
                    }
                    if (c * NMF / (TM + TN) == idx) {
                        if (c < TM) hi.x[c] = read_s(s + 2, 32 * c);
                        else hi.w[c - TM] = read_s(s + 2, L::SX + 32 * (c - TM));
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            mx_wait_lds();                                   // this stage's slot has been read
            // Scale piece g = (s + NS) / 4 + 1, ahead of the copies of stage s + NS = 4 (g - 1).
            if (((s + NS) & 3) == 0) {
                const int g = ((s + NS) >> 2) + 1;
#pragma unroll
                for (int c = 0; c < NSC; ++c) copy_s(g, (int)((uint32_t)g % L::NG), c);
            }
            Scales next;
#pragma unroll
            for (int idx = 0; idx < NMF; ++idx) {
                const int i = idx / TN, j = idx % TN;
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(B.w[j]), mx_operand(B.x[i]), acc[i][j], 4, 4,
                                                                            1, (int)now.w[j], 1, (int)now.x[i]);
#pragma unroll
                for (int c = 0; c < TM + TN; ++c)
                    if (c * NMF / (TM + TN) == idx) {
                        if (c < TM) {
                            A.x[c] = read_x(nslot, 0, c);
                            next.x[c] = pick(lo.x[c], hi.x[c], sh_x[c]);
                            lo.x[c] = hi.x[c];
                        } else {
                            A.w[c - TM] = read_w(nslot, 0, c - TM);
                            next.w[c - TM] = pick(lo.w[c - TM], hi.w[c - TM], sh_w[c - TM]);
                            lo.w[c - TM] = hi.w[c - TM];
                        }
                    }
#pragma unroll
                for (int c = 0; c < G; ++c)
                    if (c * NMF / G == idx) copy(s + NS, slot, c);
                __builtin_amdgcn_sched_barrier(0);
            }
            now = next;
            slot = nslot;
        }
        mx_wait_copies<0>();
        if (nk & 3) {
            const int left = nk & 3;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bool in = 2 * lhi + t < left;
                Step o;
                Scales sc;
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    o.x[i] = read_x(slot, t, i);
                    if (!in) o.x[i] = uint4_t{0, 0, 0, 0};
                    sc.x[i] = in ? now.x[i] >> (8 * t) : 0u;
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    o.w[j] = read_w(slot, t, j);
                    sc.w[j] = in ? now.w[j] >> (8 * t) : 0u;
                }
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(o.w[j]), mx_operand(o.x[i]), acc[i][j], 4, 4,
                                                                                    0, (int)sc.w[j], 0, (int)sc.x[i]);
            }
        }
    }
    mx_join<YT, TM, TN, WAVES, false>(acc, (float *)smem, a, tile);
}

template <typename K>
static hipError_t launch_mx_mid_k(K kernel, int lds, int waves, int BM, int BN, std::atomic<uint64_t> &done, MxMidArgs &a, hipStream_t s) {
    if (lds > 64 * 1024)
        if (hipError_t e = mx_allow_lds((const void *)kernel, lds, done)) return e;
    a.tiles_m = (a.M + BM - 1) / BM;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.tiles_m * ((a.N + BN - 1) / BN)), 1, (unsigned)a.S), dim3(64 * waves), lds, s, a);
    return hipGetLastError();
}
template <int XT, int YT, int TM, int TN, int NS, int XR, int WAVES, bool PIECES, bool EPI>
static hipError_t launch_mx_mid_t(MxMidArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    typedef MxMidLds<TM, TN, NS, XR, WAVES> L;
    static_assert(L::TOTAL <= 160 * 1024, "LDS budget");
    return launch_mx_mid_k(mx_mid_kernel<XT, YT, TM, TN, NS, XR, WAVES, PIECES, EPI>, L::TOTAL, WAVES, 32 * TM, 32 * TN, done, a, s);
}
template <int YT, int TM, int TN, int NS, int WAVES>
static hipError_t launch_mx_mid4_t(MxMidArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    typedef MxMid4Lds<TM, TN, NS, WAVES> L;
    static_assert(L::TOTAL <= 160 * 1024, "LDS budget");
    return launch_mx_mid_k(mx_mid4_kernel<YT, TM, TN, NS, WAVES>, L::TOTAL, WAVES, 32 * TM, 32 * TN, done, a, s);
}

template <int XT, int YT, bool PIECES, bool EPI>
static hipError_t launch_mx_mid_e(MxMidArgs &a, int kind, hipStream_t s) {
    // With 32 rows or fewer a stage is short, and eight waves take each other's waits; fewer rows of X
    // leave the rings more stages.
    if (kind == MX_MID_32x64)
        return a.M <= 8 ? launch_mx_mid_t<XT, YT, 1, 2, 5, 8, 8, PIECES, EPI>(a, s)
             : a.M <= 16 ? launch_mx_mid_t<XT, YT, 1, 2, 3, 16, 8, PIECES, EPI>(a, s) : launch_mx_mid_t<XT, YT, 1, 2, 5, 32, 4, PIECES, EPI>(a, s);
    if (kind == MX_MID_32x32)
        return a.M <= 8 ? launch_mx_mid_t<XT, YT, 1, 1, 8, 8, 8, PIECES, EPI>(a, s)
             : a.M <= 16 ? launch_mx_mid_t<XT, YT, 1, 1, 5, 16, 8, PIECES, EPI>(a, s) : launch_mx_mid_t<XT, YT, 1, 1, 3, 32, 8, PIECES, EPI>(a, s);
    return launch_mx_mid_t<XT, YT, 2, 2, 3, 64, 4, PIECES, EPI>(a, s);
}
template <int XT, int YT, bool PIECES>
static hipError_t launch_mx_mid_x(MxMidArgs &a, int kind, const MxEpilogue *epi, hipStream_t s) {
    if (!epi) return launch_mx_mid_e<XT, YT, PIECES, false>(a, kind, s);
    a.epi = *epi;
    return launch_mx_mid_e<XT, YT, PIECES, true>(a, kind, s);
}
template <int YT>
static hipError_t launch_mx_mid_y(MxMidArgs &a, int kind, hipStream_t s) {
    return kind == MX_MID_64x64 ? launch_mx_mid4_t<YT, 2, 2, 3, 4>(a, s) : launch_mx_mid4_t<YT, 1, 1, 3, 8>(a, s);
}

hipError_t launch_mx_mid(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s) {
    MxMidArgs a = {(const uint8_t *)c.X, c.Xs, c.Xs ? c.K / 2 : c.ldx * 2, c.W, c.Ws, c.Y, c.ldy, (int)c.M, (int)(c.K / MX_BLOCK), (int)c.N, (int)c.K * 2};
    a.units = a.row_units = (a.nb + 3) / 4;
    a.S = p.S;
    char *ws = (char *)scratch;
    a.tickets = p.S > 1 ? (uint32_t *)(ws - COUNTER_BYTES) : nullptr;
    if (!c.Xs && c.x_dt == DT_F32) {
        a.X = (const uint8_t *)ws;
        const hipError_t e = launch_mx_split(c, (uint16_t *)ws, s);
        if (e != hipSuccess) return e;
        a.kx = 3 * 128 * a.row_units * 2;
        a.ldx = a.kx;
        a.units = 3 * a.row_units;
        ws += 2 * mx_pieces(c.M, c.K);
    }
    a.part = p.S > 1 ? (float *)ws : nullptr;
    if (c.Xs)
        return c.x_dt == DT_F16 ? launch_mx_mid_y<DT_F16>(a, p.kind, s)
             : c.x_dt == DT_BF16 ? launch_mx_mid_y<DT_BF16>(a, p.kind, s) : launch_mx_mid_y<DT_F32>(a, p.kind, s);
    return c.x_dt == DT_F16 ? launch_mx_mid_x<DT_F16, DT_F16, false>(a, p.kind, c.epi, s)
         : c.x_dt == DT_BF16 ? launch_mx_mid_x<DT_BF16, DT_BF16, false>(a, p.kind, c.epi, s) : launch_mx_mid_x<DT_BF16, DT_F32, true>(a, p.kind, c.epi, s);
}

}  // namespace mcq4
