// RMS norms of the heads of q and k and the rotation of their channels, in one pass.
//
//   f = x (mean(x^2) + eps)^-1/2 w        where there is a weight
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position[axis(i)] inv_freq[i]  for pair i
//
// A lane takes eight channels of a head, four whole pairs where they are rotated: two pieces of four
// channels `half` apart, or one of eight.  So nothing but the sum of squares moves between lanes (8, 16, 32
// or 64 of them are a head), and the lane's four sines and cosines serve every head of the token.
//
// Bound by memory where there are many tokens: 8192 of 32 + 8 heads of 128, bf16, take 33 us, 5.1 TB/s where a large copy
// reaches 5.13 (29.4 of them the kernel in a trace, with inputs partly in the caches; ordinary stores, which push those out, 3 us more,
// and 7 on top while the heads of q and k stood in one row, with selects between them for each channel).  Few tokens take as long
// as the call: 4 of them 6.3 us, most of it on the host.
//
// The angle in turns is a product in fp64, taken to its part in a turn there: in fp32 an angle of
// 100000 radians would be off by 4e-3.
#include <algorithm>

#include "qk_rope.h"

namespace mcq4 {

// Four neighbouring elements.
template <int DT>
struct RopeFour {
    typedef typename mx_type<DT>::T T;
    typedef T V __attribute__((ext_vector_type(4)));
};
template <int DT, bool VEC>
__device__ __forceinline__ typename RopeFour<DT>::V rope_take(const void *p, int64_t at) {
    typedef RopeFour<DT> F;
    const typename F::T *t = (const typename F::T *)p + at;
    if constexpr (VEC) return *(const typename F::V *)t;
    typename F::V v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = t[e];
    return v;
}
template <int DT, bool VEC>
__device__ __forceinline__ void rope_put(void *p, int64_t at, const float *f) {
    typedef RopeFour<DT> F;
    typename F::T *t = (typename F::T *)p + at;
    typename F::V v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (typename F::T)f[e];
    if constexpr (VEC) __builtin_nontemporal_store(v, (typename F::V *)t);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = v[e];
}
// The weights of channels c0 .. c0 + 3 and c1 .. c1 + 3.
template <int DT>
__device__ __forceinline__ void rope_weight(const RopeHeads &x, int c0, int c1, float (&w)[8]) {
    const auto a = x.weight_vec ? rope_take<DT, true>(x.weight, c0) : rope_take<DT, false>(x.weight, c0);
    const auto b = x.weight_vec ? rope_take<DT, true>(x.weight, c1) : rope_take<DT, false>(x.weight, c1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        w[e] = (float)a[e];
        w[4 + e] = (float)b[e];
    }
}
__device__ __forceinline__ void rope_weights(const RopeHeads &x, int c0, int c1, float (&w)[8]) {
    if (!x.weight) return;
    if (x.weight_dt == DT_F32) rope_weight<DT_F32>(x, c0, c1, w);
    else if (x.weight_dt == DT_BF16) rope_weight<DT_BF16>(x, c0, c1, w);
    else rope_weight<DT_F16>(x, c0, c1, w);
}

// LG lanes a head; a wave takes 64 / LG heads of q or k of a token at a time, AT_ONCE times that in flight.
template <int DT, int LG, bool VEC, int AT_ONCE>
__global__ void __launch_bounds__(256)
qk_rope_kernel(Rope r, int waves_of_token) {
    constexpr int HW = 64 / LG;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int t = wave / waves_of_token, part = wave - t * waves_of_token;
    if (t >= r.T) return;
    const int u = lane & (LG - 1), sub = lane / LG;
    const bool here = 8 * u < r.D, turned = 4 * u < r.half;
    // The lane's channels: c0 .. c0 + 3 and c1 .. c1 + 3.
    const int c0 = turned && !r.pairs ? 4 * u : 8 * u, c1 = turned && !r.pairs ? r.half + 4 * u : 8 * u + 4;

    // Steps of HW heads: q's, then k's.
    typename RopeFour<DT>::V raw[AT_ONCE][2];
    const int q_steps = (r.q.heads + HW - 1) / HW, steps = q_steps + (r.k.heads + HW - 1) / HW;
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int s = s0 + i * waves_of_token;
            const RopeHeads &x = s < q_steps ? r.q : r.k;
            const int hd = (s < q_steps ? s : s - q_steps) * HW + sub;
            if (here && s < steps && hd < x.heads) {
                const int64_t at = t * x.token + hd * x.head;
                raw[i][0] = rope_take<DT, VEC>(x.x, at + c0);
                raw[i][1] = rope_take<DT, VEC>(x.x, at + c1);
            }
        }
    };
    load(part);

    float qw[8], kw[8], cs[4], sn[4];
    if (here) {
        rope_weights(r.q, c0, c1, qw);
        rope_weights(r.k, c0, c1, kw);
    }
    if (turned) {
        const float4_t freq = *(const float4_t *)(r.inv_freq + 4 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 4 * u + e;
            int axis = 0;
#pragma unroll
            for (int a = 0; a < ROPE_AXES - 1; ++a) axis += i >= r.end[a];
            const int pos = r.positions[axis * r.axis_stride + t];
            const double turns = (double)pos * ((double)freq[e] * 0.15915494309189533577);
            sincospif((float)(2.0 * (turns - rint(turns))), &sn[e], &cs[e]);
        }
    }
    const float over = 1.0f / (float)r.D;
    for (int s0 = part; s0 < steps; s0 += AT_ONCE * waves_of_token) {
        float f[AT_ONCE][8];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i][e] = (float)raw[i][e / 4][e % 4];
        if (s0 + AT_ONCE * waves_of_token < steps) load(s0 + AT_ONCE * waves_of_token);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int s = s0 + i * waves_of_token;
            if (s >= steps) break;
            const RopeHeads &x = s < q_steps ? r.q : r.k;
            const int hd = (s < q_steps ? s : s - q_steps) * HW + sub;
            const bool ok = here && hd < x.heads;
            if (x.weight) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += f[i][e] * f[i][e];
                ss = ok ? ss : 0.f;
#pragma unroll
                for (int d = 1; d < LG; d <<= 1) ss += __shfl_xor(ss, d);
                const float rstd = rsqrtf(ss * over + r.eps);
                if (s < q_steps) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * rstd * qw[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * rstd * kw[e];
                }
            }
            if (turned) {
                if (r.pairs) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = f[i][2 * e], b = f[i][2 * e + 1];
                        f[i][2 * e] = a * cs[e] - b * sn[e];
                        f[i][2 * e + 1] = b * cs[e] + a * sn[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = f[i][e], b = f[i][e + 4];
                        f[i][e] = a * cs[e] - b * sn[e];
                        f[i][e + 4] = b * cs[e] + a * sn[e];
                    }
                }
            }
            if (ok) {
                const int64_t at = t * x.y_token + hd * x.y_head;
                rope_put<DT, VEC>(x.y, at + c0, f[i]);
                rope_put<DT, VEC>(x.y, at + c1, f[i] + 4);
            }
        }
    }
}

template <int DT, int LG, bool VEC>
static hipError_t launch_qk_rope_t(const Rope &r, hipStream_t s) {
    const int hw = 64 / LG, steps = (r.q.heads + hw - 1) / hw + (r.k.heads + hw - 1) / hw;
    // A token's sines are made once for a wave, so a token is one wave's where that fills the card, 32 waves a CU (2560 tokens
    // of 128 heads of 64, fp32: 29.7 us with three waves a token, 33.0 with one; 2501 of 32 of 80, fp16: 11.6 and 11.1).
    const int waves = std::max(1, std::min(steps, 8192 / r.T)), each = (steps + waves - 1) / waves;
    const dim3 grid((unsigned)(((int64_t)r.T * waves + 3) / 4)), block(256);
    constexpr int MOST = DT == DT_F32 ? 3 : 5;
    if (each == 1) hipLaunchKernelGGL((qk_rope_kernel<DT, LG, VEC, 1>), grid, block, 0, s, r, waves);
    else if (each == 2) hipLaunchKernelGGL((qk_rope_kernel<DT, LG, VEC, 2>), grid, block, 0, s, r, waves);
    else hipLaunchKernelGGL((qk_rope_kernel<DT, LG, VEC, MOST>), grid, block, 0, s, r, waves);
    return hipGetLastError();
}
template <int DT, bool VEC>
static hipError_t launch_qk_rope_v(const Rope &r, hipStream_t s) {
    return r.D <= 64 ? launch_qk_rope_t<DT, 8, VEC>(r, s) : r.D <= 128 ? launch_qk_rope_t<DT, 16, VEC>(r, s)
         : r.D <= 256 ? launch_qk_rope_t<DT, 32, VEC>(r, s) : launch_qk_rope_t<DT, 64, VEC>(r, s);
}
template <int DT>
static hipError_t launch_qk_rope_d(const Rope &r, hipStream_t s) { return r.vec ? launch_qk_rope_v<DT, true>(r, s) : launch_qk_rope_v<DT, false>(r, s); }

hipError_t launch_qk_rope(const Rope &r, hipStream_t s) {
    return r.dt == DT_F32 ? launch_qk_rope_d<DT_F32>(r, s) : r.dt == DT_BF16 ? launch_qk_rope_d<DT_BF16>(r, s) : launch_qk_rope_d<DT_F16>(r, s);
}

}  // namespace mcq4
