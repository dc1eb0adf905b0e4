// Products with MXFP4 weights, operands straight from memory to registers:
// Y[M, N] = X[M, K] W[N, K]^T for few rows.
//
// A wave computes 16 columns (A operand: 16 rows of W) times 16 rows of X (B operand).  One
// 16-byte load gives a lane one block of its row; lane l holds row l % 16 and, of four
// consecutive blocks, block l / 16.  The order in which a product runs over K is free as long
// as both operands agree, so MFMA j of a step takes bytes 4 j .. 4 j + 3 of every lane's block
// and X's elements 8 j .. 8 j + 7 of the same block: no operand is ever moved between lanes.
// The waves of a workgroup share out K and add their sums in LDS, in wave order.
//
// 16-bit X: weights converted to X's type, v_mfma_f32_16x16x32.  fp32 X: three bf16 pieces
// whose sum is the value, with the exact bf16 weights.  Microscaled X: v_mfma_scale_f32_16x16x128 on both packed blocks.
//
// Bound by latency: 1 x 4096 x 4096 takes 5.4 us, of which an empty launch is 1.7, the loads (all
// of a wave's in flight at once) 2 and the waves' sum the rest; 8.9 MB alone would take 1.8.
#include <algorithm>

#include "mx_gemm.h"

namespace mcq4 {

constexpr int MXD_WAVES = 16;

struct MxDirectArgs {
    const uint8_t *X, *Xs;
    int64_t ldx;                   // bytes
    const uint8_t *W, *Ws;
    void *Y;
    int64_t ldy;
    int M, nb, N;
    MxEpilogue epi;
};

// XT: type of X, of Y where XQ (microscaled X).  U steps' loads go out before the first of them is
// used: a wave has at most a few steps, and the latency of its loads is what the call takes.
template <int XT, bool XQ, int U, bool EPI>
__global__ void __launch_bounds__(64 * MXD_WAVES)
mx_direct_kernel(MxDirectArgs a) {
    __shared__ float4_t part[MXD_WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int row = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int n = min(n0 + row, a.N - 1), m = min(m0 + row, a.M - 1);
    const uint8_t *w = a.W + (int64_t)n * a.nb * 16, *ws = a.Ws + (int64_t)n * a.nb;
    const uint8_t *x = a.X + m * a.ldx, *xs = XQ ? a.Xs + (int64_t)m * a.nb : nullptr;
    constexpr int XV = XQ ? 1 : XT == DT_F32 ? 8 : 4;         // 16-byte pieces of X per block
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    MxOperands<XT, 4> ops;                                    // on their way during the product
    if constexpr (EPI)
        if (wave == 0) ops.load(a.epi, m0 + row, n0 + 4 * g, a.M, a.N);
    for (int b0 = 4 * wave; b0 < a.nb; b0 += 4 * waves * U) {
        uint4_t q[U], xv[U][XV];
        uint32_t sb[U], xb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = min(b0 + 4 * waves * u + g, a.nb - 1);
            q[u] = *(const uint4_t *)(w + (int64_t)kb * 16);
            sb[u] = ws[kb];
#pragma unroll
            for (int j = 0; j < XV; ++j) xv[u][j] = *(const uint4_t *)(x + ((int64_t)kb * XV + j) * 16);
            if constexpr (XQ) xb[u] = xs[kb];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (b0 + 4 * waves * u >= a.nb) break;
            if (b0 + 4 * waves * u + g >= a.nb) {             // past the last block: zeros and a finite scale
                q[u] = uint4_t{0, 0, 0, 0};
                sb[u] = xb[u] = 0;
#pragma unroll
                for (int j = 0; j < XV; ++j) xv[u][j] = uint4_t{0, 0, 0, 0};
            }
            if constexpr (XQ) {
                acc = mx_mfma16_fp4(q[u], xv[u][0], acc, sb[u], xb[u]);
            } else {
                const float s = mx_scale(sb[u]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (XT == DT_F32) {
                        const float4_t f0 = bitcast<float4_t>(xv[u][2 * j]), f1 = bitcast<float4_t>(xv[u][2 * j + 1]);
                        const float f[8] = {f0[0], f0[1], f0[2], f0[3], f1[0], f1[1], f1[2], f1[3]};
                        const uint4_t wv = mx_weights8<DT_BF16>(q[u][j], s);
                        uint4_t pc[3];
                        mx_split8(f, pc);
#pragma unroll
                        for (int t = 2; t >= 0; --t) acc = mx_mfma16<DT_BF16>(wv, pc[t], acc);
                    } else {
                        acc = mx_mfma16<XT>(mx_weights8<XT>(q[u][j], s), xv[u][j], acc);
                    }
                }
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    for (int i = 1; i < waves; ++i) acc += part[i][lane];
    // D of the MFMA: lane l holds columns n0 + 4 (l / 16) .. + 3 of Y's row m0 + l % 16.
    if (m0 + row >= a.M) return;
    if constexpr (EPI) {
        float v[4] = {acc[0], acc[1], acc[2], acc[3]};
        mx_finish<XT, 4>(a.epi, ops, v);
        acc = float4_t{v[0], v[1], v[2], v[3]};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + 4 * g + i < a.N) mx_store<XT>(a.Y, (int64_t)(m0 + row) * a.ldy + n0 + 4 * g + i, acc[i]);
}

// Four waves at least where there are as many steps of four blocks, and up to four steps each.
int mx_direct_waves(int64_t K) {
    const int64_t steps = (K / MX_BLOCK + 3) / 4;
    return (int)std::max<int64_t>(std::min<int64_t>(steps, 4), std::min<int64_t>(MXD_WAVES, (steps + 3) / 4));
}
int mx_direct_batch(const MxCall &c) { return !c.Xs && c.x_dt == DT_F32 ? 2 : 4; }

hipError_t launch_mx_direct(const MxCall &c, hipStream_t s) {
    const int es = c.x_dt == DT_F32 ? 4 : 2;
    MxDirectArgs a = {(const uint8_t *)c.X, c.Xs, c.Xs ? c.ldx : c.ldx * es, c.W, c.Ws, c.Y, c.ldy, (int)c.M, (int)(c.K / MX_BLOCK), (int)c.N, {}};
    const dim3 grid((unsigned)((c.N + 15) / 16), (unsigned)((c.M + 15) / 16)), block(64 * mx_direct_waves(c.K));
    if (c.Xs) {
        if (c.x_dt == DT_F16) hipLaunchKernelGGL((mx_direct_kernel<DT_F16, true, 4, false>), grid, block, 0, s, a);
        else if (c.x_dt == DT_BF16) hipLaunchKernelGGL((mx_direct_kernel<DT_BF16, true, 4, false>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((mx_direct_kernel<DT_F32, true, 4, false>), grid, block, 0, s, a);
    } else if (c.epi) {
        a.epi = *c.epi;
        if (c.x_dt == DT_F16) hipLaunchKernelGGL((mx_direct_kernel<DT_F16, false, 4, true>), grid, block, 0, s, a);
        else if (c.x_dt == DT_BF16) hipLaunchKernelGGL((mx_direct_kernel<DT_BF16, false, 4, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((mx_direct_kernel<DT_F32, false, 2, true>), grid, block, 0, s, a);
    } else {
        if (c.x_dt == DT_F16) hipLaunchKernelGGL((mx_direct_kernel<DT_F16, false, 4, false>), grid, block, 0, s, a);
        else if (c.x_dt == DT_BF16) hipLaunchKernelGGL((mx_direct_kernel<DT_BF16, false, 4, false>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((mx_direct_kernel<DT_F32, false, 2, false>), grid, block, 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace mcq4
