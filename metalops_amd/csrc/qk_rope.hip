// RMS norms of the heads of q and k and the rotation of their channels, in one pass.
//
//   f = x (mean(x^2) + eps)^-1/2 w        where there is a weight
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position[axis(i)] inv_freq[i]  for pair i
//
// A lane takes eight channels of a head, four whole pairs where they are rotated: two pieces of four
// channels `half` apart, or one of eight.  So nothing but the sum of squares moves between lanes (8, 16, 32
// or 64 of them are a head), and the lane's four sines and cosines serve every head of the token.
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
    if constexpr (VEC) *(typename F::V *)t = v;
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = v[e];
}
__device__ __forceinline__ void rope_weight(const RopeHeads &x, int c0, int c1, float (&w)[8]) {
    if (!x.weight) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = e < 4 ? c0 + e : c1 + e - 4;
        w[e] = x.weight_dt == DT_F32 ? ((const float *)x.weight)[c]
             : x.weight_dt == DT_BF16 ? (float)((const __bf16 *)x.weight)[c] : (float)((const _Float16 *)x.weight)[c];
    }
}

// LG lanes a head; a wave takes 64 / LG heads of a token at a time, AT_ONCE times that in flight.
template <int DT, int LG, bool VEC>
__global__ void __launch_bounds__(256)
qk_rope_kernel(Rope r, int waves_of_token) {
    constexpr int HW = 64 / LG, AT_ONCE = DT == DT_F32 ? 3 : 5;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int t = wave / waves_of_token, part = wave - t * waves_of_token;
    if (t >= r.T) return;
    const int u = lane & (LG - 1), heads = r.q.heads + r.k.heads;
    const bool here = 8 * u < r.D, turned = 4 * u < r.half;
    // The lane's channels: c0 .. c0 + 3 and c1 .. c1 + 3.
    const int c0 = turned && !r.pairs ? 4 * u : 8 * u, c1 = turned && !r.pairs ? r.half + 4 * u : 8 * u + 4;

    typename RopeFour<DT>::V raw[AT_ONCE][2];
    const int steps = (heads + HW - 1) / HW;
    auto place = [&](int s, bool &ok) {
        const int hd = s * HW + lane / LG;
        ok = here && s < steps && hd < heads;
        return hd;
    };
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            bool ok;
            const int hd = place(s0 + i * waves_of_token, ok);
            const bool is_k = hd >= r.q.heads;
            const void *x = is_k ? r.k.x : r.q.x;
            const int64_t at = is_k ? t * r.k.token + (hd - r.q.heads) * r.k.head : t * r.q.token + hd * r.q.head;
            if (ok) {
                raw[i][0] = rope_take<DT, VEC>(x, at + c0);
                raw[i][1] = rope_take<DT, VEC>(x, at + c1);
            }
        }
    };
    load(part);

    float qw[8], kw[8], cs[4], sn[4];
    if (here) {
        rope_weight(r.q, c0, c1, qw);
        rope_weight(r.k, c0, c1, kw);
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
            bool ok;
            const int hd = place(s0 + i * waves_of_token, ok);
            const bool is_k = hd >= r.q.heads;
            if (is_k ? r.k.weight != nullptr : r.q.weight != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += f[i][e] * f[i][e];
                ss = ok ? ss : 0.f;
#pragma unroll
                for (int d = 1; d < LG; d <<= 1) ss += __shfl_xor(ss, d);       // of a head's lanes, which take one branch
                const float rstd = rsqrtf(ss * over + r.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * rstd * (is_k ? kw[e] : qw[e]);
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
                void *y = is_k ? r.k.y : r.q.y;
                const int64_t at = is_k ? t * r.k.y_token + (hd - r.q.heads) * r.k.y_head : t * r.q.y_token + hd * r.q.y_head;
                rope_put<DT, VEC>(y, at + c0, f[i]);
                rope_put<DT, VEC>(y, at + c1, f[i] + 4);
            }
        }
    }
}

template <int DT, int LG, bool VEC>
static hipError_t launch_qk_rope_t(const Rope &r, hipStream_t s) {
    const int steps = (r.q.heads + r.k.heads + 64 / LG - 1) / (64 / LG);
    // A token's sines are made once for a wave, so a token is a wave's where that fills the card (8 waves a CU).
    const int waves = std::max(1, std::min(steps, 2048 / r.T));
    hipLaunchKernelGGL((qk_rope_kernel<DT, LG, VEC>), dim3((unsigned)(((int64_t)r.T * waves + 3) / 4)), dim3(256), 0, s, r, waves);
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
