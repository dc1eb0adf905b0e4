// Shared parts of the LDS-staged MXFP4 products (mx_gemm.hip, mx_gemm4.hip): tile order,
// copies to LDS, the store of a tile and the sum of K splits.
#pragma once

#include <algorithm>
#include <atomic>

#include "mx_common.h"

namespace mcq4 {

struct MxTile { int m, n; };
// Workgroup i of a grid runs on XCD i % 8: each XCD gets consecutive tiles, row tiles
// first, so that its L2 serves a strip of weights to all row tiles.
__device__ __forceinline__ MxTile mx_tile(int tiles_m) {
    const int bid = blockIdx.x, gx = gridDim.x, xcd = bid & 7, q = gx >> 3, r = gx & 7;
    const int t = xcd * q + min(xcd, r) + (bid >> 3);
    return {t % tiles_m, t / tiles_m};
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rsrc(const void *p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, (int)max((int64_t)0, bytes), 0x00020000);
}
// 64 lanes times 16 (or 4) bytes to LDS at dst, in lane order; 0 past the resource's end.
__device__ __forceinline__ void mx_copy16(__amdgpu_buffer_rsrc_t rs, uint8_t *dst, int vo, int so) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)dst, 16, vo, so, 0, 0);
}
__device__ __forceinline__ void mx_copy4(__amdgpu_buffer_rsrc_t rs, uint8_t *dst, int vo, int so) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)dst, 4, vo, so, 0, 0);
}
typedef __attribute__((address_space(3))) uint4_t lds_uint4;
typedef __attribute__((address_space(3))) uint2_t lds_uint2;
__device__ __forceinline__ uint4_t mx_lds16(uint32_t addr) { return *(const lds_uint4 *)lds_ptr(addr); }
__device__ __forceinline__ uint32_t mx_lds4(uint32_t addr) { return *(const lds_u32 *)lds_ptr(addr); }

template <int DT>
__device__ __forceinline__ uint32_t mx_pair(float a, float b) {
    if constexpr (DT == DT_BF16) return bitcast<uint32_t>(__builtin_convertvector((float2_t{a, b}), bf16x2_t));
    else return bitcast<uint32_t>(half2_t{(_Float16)a, (_Float16)b});
}

// ---- what follows the product (MxEpilogue), W neighbouring columns of a row at a time ----

template <int DT, int W>
struct mx_vec { typedef typename mx_type<DT>::T T __attribute__((ext_vector_type(W))); };

// W elements from p, as many of them as `left`; in one piece where `vec`.
template <int DT, int W>
__device__ __forceinline__ typename mx_vec<DT, W>::T mx_take(const void *p, int64_t at, int left, bool vec) {
    typedef typename mx_type<DT>::T T;
    typedef typename mx_vec<DT, W>::T V;
    const T *t = (const T *)p + at;
    if (vec && left >= W) return *(const V *)t;
    V v;
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = e < left ? t[e] : (T)0.f;
    return v;
}

// The operands of an epilogue for columns n .. of row m; loaded ahead of their use, as they lie in memory.
template <int DT, int W>
struct MxOperands {
    typename mx_vec<DT, W>::T mul, res;
    float bias[W];
    __device__ __forceinline__ void load(const MxEpilogue &e, int m, int n, int M, int N) {
        load_rows(e, m, n, M, N);
        load_bias(e, n, N);
    }
    __device__ __forceinline__ void load_rows(const MxEpilogue &e, int m, int n, int M, int N) {
        if (m >= M || n >= N) return;
        if (e.mul) mul = mx_take<DT, W>(e.mul, (int64_t)m * e.ld_mul + n, N - n, e.vec);
        if (e.res) res = mx_take<DT, W>(e.res, (int64_t)m * e.ld_res + n, N - n, e.vec);
    }
    __device__ __forceinline__ void load_bias(const MxEpilogue &e, int n, int N) {
        if (e.bias && n < N) {
            if (DT == DT_F32 || e.bias_dt == DT_F32) {
                const auto b = mx_take<DT_F32, W>(e.bias, n, N - n, e.vec);
#pragma unroll
                for (int i = 0; i < W; ++i) bias[i] = b[i];
            } else {
                const auto b = mx_take<DT, W>(e.bias, n, N - n, e.vec);
#pragma unroll
                for (int i = 0; i < W; ++i) bias[i] = (float)b[i];
            }
        }
    }
};

// 1 / (1 + e^-x).  16-bit results take the exponential and the reciprocal of the VALU: off by 2^-19 at most for x from
// -16 on, below which x / (1 + e^-x) is no more than 2e-6.
template <int DT>
__device__ __forceinline__ float mx_sigmoid(float x) {
    if constexpr (DT == DT_F32) return 1.0f / (1.0f + expf(-x));
    else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}
// x Phi(x).  16-bit results: erfc(z) / 2 = (c1 t + .. + c8 t^8) e^(-z^2) with t = 1 / (1 + p z) and z = |x| / sqrt 2, the form of
// Abramowitz and Stegun 7.1.26.  The c are fitted to e^(z^2) erfc(z) / 2 for z from 0 to 9.6, where results leave bf16's range, with
// the error relative to it, 2^-23 (weighted least squares, the weights raised where the error is largest): so the left tail keeps its digits
// too.  All in all off by 2^-20 of the result down to -3, 2^-18 to -8 and 2^-16 to -13, where the exponent's rounding is what counts;
// with the five published terms, whose error is small against erfc(0) only, by 2^-11 to -4, 2^-9 to -5 and 4% to -13.
// 2048 x 4096 x 14336 with gelu takes 227.5 us, 227 with five terms; erfcf took 48 us more.  fp32: erfcf.
template <int DT>
__device__ __forceinline__ float mx_gelu(float x) {
    if constexpr (DT == DT_F32) return x * (0.5f * erfcf(-0.70710678118654752f * x));
    else {
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678f, fabsf(x), 1.0f));
        float s = __builtin_fmaf(-0.0707279667f, t, 0.248994008f);
        s = __builtin_fmaf(s, t, -0.204001158f);
        s = __builtin_fmaf(s, t, 0.227509022f);
        s = __builtin_fmaf(s, t, 0.0122911232f);
        s = __builtin_fmaf(s, t, 0.103058256f);
        s = __builtin_fmaf(s, t, 0.0903494805f);
        s = __builtin_fmaf(s, t, 0.0925272852f);
        const float half = s * t * __builtin_amdgcn_exp2f(-0.72134752044448170f * x * x);             // erfc(z) / 2
        return x * (x < 0.f ? half : 1.0f - half);
    }
}
template <int DT, int W>
__device__ __forceinline__ void mx_finish(const MxEpilogue &e, const MxOperands<DT, W> &o, const float (&bias)[W], float (&v)[W]) {
    if (e.bias)
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += bias[i];
    switch (e.act) {
        case MX_ACT_RELU:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];      // NaN stays
            break;
        case MX_ACT_SILU:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] *= mx_sigmoid<DT>(v[i]);
            break;
        case MX_ACT_GELU:
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = mx_gelu<DT>(v[i]);
            break;
        case MX_ACT_GELU_TANH:                   // x / 2 (1 + tanh u) = x sigmoid(2 u)
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] *= mx_sigmoid<DT>(1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]));
            break;
        default: break;
    }
    if (e.mul)
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] *= (float)o.mul[i];
    if (e.res)
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += (float)o.res[i];
}

template <int DT, int W>
__device__ __forceinline__ void mx_finish(const MxEpilogue &e, const MxOperands<DT, W> &o, float (&v)[W]) { mx_finish<DT, W>(e, o, o.bias, v); }

// A sum that is read from here on only.  Sums of 16 tiles fill the accumulation registers, and the compiler copies all
// of them ahead of the stores, more than there are registers for.
template <int TILES>
__device__ __forceinline__ float16_t mx_from_here(float16_t x) {
    if constexpr (TILES >= 16) asm volatile("" : "+a"(x));
    return x;
}

// A wave's TM x TN results of v_mfma_f32_32x32 with the weights as the A operand: lane l
// holds row 32 i + l % 32 and, in register r, column 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.
// 16-bit results go through the wave's own LDS, [32 TM][64 TN + 16 bytes], so that a row's
// 64 TN bytes are stored in one piece; fp32 ones are stored four columns at a time.
template <int DT, int TM, int TN>
__device__ __forceinline__ void mx_store_tile(const float16_t (&acc)[TM][TN], uint8_t *lds, void *Y, int64_t ldy, int m0, int n0,
                                              int M, int N) {
    const int lane = threadIdx.x & 63, row = lane & 31, hi = lane >> 5;
    if constexpr (DT == DT_F32) {
        const bool vec = (ldy & 3) == 0 && ((uintptr_t)Y & 15) == 0;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const float16_t t = mx_from_here<TM * TN>(acc[i][j]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = m0 + 32 * i + row, n = n0 + 32 * j + 8 * q + 4 * hi;
                    if (m >= M || n >= N) continue;
                    float *y = (float *)Y + (int64_t)m * ldy + n;
                    const float4_t v = {t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]};
                    if (vec && n + 4 <= N) *(float4_t *)y = v;
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n + e < N) y[e] = v[e];
                }
            }
    } else {
        constexpr int PITCH = 64 * TN + 16;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const float16_t t = mx_from_here<TM * TN>(acc[i][j]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint2_t v = {mx_pair<DT>(t[4 * q], t[4 * q + 1]), mx_pair<DT>(t[4 * q + 2], t[4 * q + 3])};
                    *(uint2_t *)(lds + (32 * i + row) * PITCH + 64 * j + 16 * q + 8 * hi) = v;
                }
            }
        __builtin_amdgcn_wave_barrier();
        const bool vec = (ldy & 7) == 0 && ((uintptr_t)Y & 15) == 0;
        constexpr int LANES = 4 * TN;                     // 16 bytes each
#pragma unroll 4
        for (int p = lane; p < 32 * TM * LANES; p += 64) {
            const int m = m0 + p / LANES, n = n0 + 8 * (p % LANES);
            if (m >= M || n >= N) continue;
            const uint4_t v = *(const uint4_t *)(lds + (p / LANES) * PITCH + 16 * (p % LANES));
            uint16_t *y = (uint16_t *)Y + (int64_t)m * ldy + n;
            if (vec && n + 8 <= N) *(uint4_t *)y = v;
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + e < N) y[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
        }
    }
}
// The same with an epilogue, for any type: the sums of 32 GI rows at a time go through the wave's own LDS in fp32,
// [32 GI][128 TN + 16 bytes], so that a lane takes eight neighbouring columns of a row, whose operands and result are
// whole 16-byte pieces, and the epilogue stands in one loop.
template <int TM, int TN>
constexpr int mx_epi_rows() { return TM * TN > 2 ? TM / TN : TM; }
template <int TM, int TN>
constexpr int mx_epi_lds() { return 32 * mx_epi_rows<TM, TN>() * (128 * TN + 16); }
template <int DT, int TM, int TN>
__device__ __forceinline__ void mx_store_epi(const float16_t (&acc)[TM][TN], uint8_t *lds, const MxEpilogue &epi, void *Y, int64_t ldy, int m0, int n0,
                                             int M, int N) {
    constexpr int GI = mx_epi_rows<TM, TN>(), PITCH = 128 * TN + 16, LANES = 4 * TN;
    typedef typename mx_type<DT>::T T;
    typedef typename mx_vec<DT, 8>::T V;
    const int lane = threadIdx.x & 63, row = lane & 31, hi = lane >> 5;
    const bool vec = ldy * sizeof(T) % 16 == 0 && ((uintptr_t)Y & 15) == 0;
    // Rows of a lane's pieces lie 64 / LANES apart, its columns stay.  AT_ONCE pieces' operands are in flight while as many are
    // finished (loaded only before their use they took 32 us of 2048 x 4096 x 14336 with a gate).
    constexpr int STEPS = 32 * GI * LANES / 64, AT_ONCE = std::min(STEPS, DT == DT_F32 ? 4 : 8), BATCHES = STEPS / AT_ONCE;
    static_assert(STEPS % AT_ONCE == 0, "whole batches");
    const int n = n0 + 8 * (lane % LANES), m_lane = m0 + lane / LANES;
    MxOperands<DT, 8> own, cur[AT_ONCE], next[AT_ONCE];
    own.load_bias(epi, n, N);
    auto fetch = [&](MxOperands<DT, 8> (&o)[AT_ONCE], int batch) {
#pragma unroll
        for (int s = 0; s < AT_ONCE; ++s) o[s].load_rows(epi, m_lane + (batch * AT_ONCE + s) * (64 / LANES), n, M, N);
    };
    fetch(cur, 0);
#pragma unroll
    for (int i0 = 0; i0 < TM; i0 += GI) {
#pragma unroll
        for (int i = 0; i < GI; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const float16_t t = mx_from_here<TM * TN>(acc[i0 + i][j]);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(float4_t *)(lds + (32 * i + row) * PITCH + 128 * j + 32 * q + 16 * hi) = float4_t{t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]};
            }
        __builtin_amdgcn_wave_barrier();
        for (int b = 0; b < BATCHES; ++b) {
            const int batch = i0 / GI * BATCHES + b;
            if (batch + 1 < TM / GI * BATCHES) fetch(next, batch + 1);
            if (n < N)
#pragma unroll
                for (int s = 0; s < AT_ONCE; ++s) {
                    const int at = lane / LANES + (b * AT_ONCE + s) * (64 / LANES), m = m0 + 32 * i0 + at;
                    if (m >= M) continue;
                    const float4_t *f = (const float4_t *)(lds + at * PITCH + 32 * (lane % LANES));
                    float v[8] = {f[0][0], f[0][1], f[0][2], f[0][3], f[1][0], f[1][1], f[1][2], f[1][3]};
                    mx_finish<DT, 8>(epi, cur[s], own.bias, v);
                    T *y = (T *)Y + (int64_t)m * ldy + n;
                    if (vec && n + 8 <= N) {
                        V r;
#pragma unroll
                        for (int e = 0; e < 8; ++e) r[e] = (T)v[e];
                        *(V *)y = r;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (n + e < N) y[e] = (T)v[e];
                    }
                }
#pragma unroll
            for (int s = 0; s < AT_ONCE; ++s) cur[s] = next[s];
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <int DT, int TM, int TN>
constexpr int mx_store_lds() { return DT == DT_F32 ? 0 : 32 * TM * (64 * TN + 16); }

// fp32 partial sums of a K split, [M][ldp] with ldp = N rounded up to 4: the same lanes' columns.
template <int TM, int TN>
__device__ __forceinline__ void mx_store_part(const float16_t (&acc)[TM][TN], float *part, int64_t ldp, int m0, int n0, int M, int N) {
    const int lane = threadIdx.x & 63, row = lane & 31, hi = lane >> 5;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = m0 + 32 * i + row, n = n0 + 32 * j + 8 * q + 4 * hi;
                if (m < M && n < N)
                    *(float4_t *)(part + (int64_t)m * ldp + n) = float4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            }
}

inline int64_t mx_ldp(int64_t N) { return (N + 3) / 4 * 4; }
// Adds S partials [S][M][ldp] in order and stores them in type dt, `epi` (or null) before (mx_gemm.hip).
hipError_t launch_mx_sum(const float *part, int S, void *Y, int64_t ldy, int dt, int64_t M, int64_t N, const MxEpilogue *epi, hipStream_t s);

enum { MX_DIRECT = 0, MX_256x256 = 1, MX_128x256 = 2, MX_128x128 = 3, MX_64x128 = 4, MX_MID_64x64 = 5, MX_MID_32x64 = 6, MX_MID_32x32 = 7, MX_KINDS };
// Elements of fp32 X's three pieces, a whole number of 16 bytes.
inline int64_t mx_pieces(int64_t M, int64_t K) { return M * 3 * ((K + 127) / 128 * 128); }
hipError_t launch_mx_gemm(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s);      // 16-bit and fp32 X
hipError_t launch_mx_gemm4(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s);     // microscaled X
hipError_t launch_mx_mid(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s);       // either
// Waves of the direct kernel, and steps whose loads they send out together.
int mx_direct_waves(int64_t K);
int mx_direct_batch(const MxCall &c);
// fp32 X to three bf16 pieces, [M][3][K rounded up to 128].
hipError_t launch_mx_split(const MxCall &c, uint16_t *out, hipStream_t s);

// Once for each device: `kernel` may use `lds` bytes.
inline hipError_t mx_allow_lds(const void *kernel, int lds, std::atomic<uint64_t> &done) {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return hipSuccess;
    if (hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds)) return e;
    done.fetch_or(bit, std::memory_order_acq_rel);
    return hipSuccess;
}

}  // namespace mcq4
