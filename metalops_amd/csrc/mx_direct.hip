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
#include <algorithm>

#include "mx_common.h"

namespace mcq4 {

constexpr int MXD_WAVES = 8;

struct MxDirectArgs {
    const uint8_t *X, *Xs;
    int64_t ldx;                   // bytes
    const uint8_t *W, *Ws;
    void *Y;
    int64_t ldy;
    int M, nb, N;
};

// XT: type of X, of Y where XQ (microscaled X).
template <int XT, bool XQ>
__global__ void __launch_bounds__(64 * MXD_WAVES)
mx_direct_kernel(MxDirectArgs a) {
    __shared__ float4_t part[MXD_WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int row = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int n = min(n0 + row, a.N - 1), m = min(m0 + row, a.M - 1);
    const uint8_t *w = a.W + (int64_t)n * a.nb * 16, *ws = a.Ws + (int64_t)n * a.nb;
    const uint8_t *x = a.X + m * a.ldx;
    constexpr int XB = XQ ? 16 : XT == DT_F32 ? 128 : 64;     // bytes of X per block
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int b = 4 * wave + g; b - g < a.nb; b += 4 * waves) {
        const bool in = b < a.nb;
        const int kb = in ? b : a.nb - 1;
        uint4_t q = *(const uint4_t *)(w + kb * 16);
        const uint32_t sb = ws[kb];
        if constexpr (XQ) {
            uint4_t xq = *(const uint4_t *)(x + kb * 16);
            const uint32_t xs = a.Xs[(int64_t)m * a.nb + kb];
            // Past the last block: zero elements and a finite scale.
            if (!in) { q = uint4_t{0, 0, 0, 0}; xq = q; }
            acc = mx_mfma16_fp4(q, xq, acc, in ? sb : 0u, in ? xs : 0u);
        } else {
            const float s = mx_scale(in ? sb : 0u);
            if (!in) q = uint4_t{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (XT == DT_F32) {
                    const float4_t *p = (const float4_t *)(x + (int64_t)kb * XB + 32 * j);
                    const float4_t u = p[0], v = p[1];
                    const float f[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                    const uint4_t wv = mx_weights8<DT_BF16>(q[j], s);
                    uint4_t pc[3];
                    mx_split8(f, pc);
#pragma unroll
                    for (int t = 2; t >= 0; --t) acc = mx_mfma16<DT_BF16>(wv, in ? pc[t] : uint4_t{0, 0, 0, 0}, acc);
                } else {
                    const uint4_t xv = *(const uint4_t *)(x + (int64_t)kb * XB + 16 * j);
                    acc = mx_mfma16<XT>(mx_weights8<XT>(q[j], s), in ? xv : uint4_t{0, 0, 0, 0}, acc);
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
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + 4 * g + i < a.N) mx_store<XT>(a.Y, (int64_t)(m0 + row) * a.ldy + n0 + 4 * g + i, acc[i]);
}

hipError_t launch_mx_direct(const MxCall &c, hipStream_t s) {
    const int es = c.x_dt == DT_F32 ? 4 : 2;
    MxDirectArgs a = {(const uint8_t *)c.X, c.Xs, c.Xs ? c.ldx : c.ldx * es, c.W, c.Ws, c.Y, c.ldy, (int)c.M, (int)(c.K / MX_BLOCK), (int)c.N};
    const int waves = std::max(1, std::min(MXD_WAVES, (a.nb + 3) / 4));
    const dim3 grid((unsigned)((c.N + 15) / 16), (unsigned)((c.M + 15) / 16)), block(64 * waves);
    if (c.Xs) {
        if (c.x_dt == DT_F16) hipLaunchKernelGGL((mx_direct_kernel<DT_F16, true>), grid, block, 0, s, a);
        else if (c.x_dt == DT_BF16) hipLaunchKernelGGL((mx_direct_kernel<DT_BF16, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((mx_direct_kernel<DT_F32, true>), grid, block, 0, s, a);
    } else {
        if (c.x_dt == DT_F16) hipLaunchKernelGGL((mx_direct_kernel<DT_F16, false>), grid, block, 0, s, a);
        else if (c.x_dt == DT_BF16) hipLaunchKernelGGL((mx_direct_kernel<DT_BF16, false>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((mx_direct_kernel<DT_F32, false>), grid, block, 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace mcq4
