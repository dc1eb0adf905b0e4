// Shared parts of the microscaled kernels (mx_*.hip, kv8_*.hip).
//
// MXFP4 (OCP Microscaling Formats v1.0): blocks of 32 consecutive K elements of a row; a
// scale byte b stands for 2^(b - 127), 255 for NaN; an element is e2m1 (0, 0.5, 1, 1.5, 2,
// 3, 4, 6 and their negatives).  packed[R][K/2]: element 2i in the low nibble of byte i,
// 2i + 1 in the high one; scales[R][K/32].  A block's 16 bytes are one 16-byte load and,
// as they stand, one lane's operand of the scaled MFMA.
#pragma once

#include "q4_prefill.h"

namespace mcq4 {

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

constexpr int MX_BLOCK = 32;

// The fp32 scale operand of the v_cvt_scalef32_* instructions for a scale byte.  They use
// the exponent field alone, except that an exponent of 255 with a mantissa is NaN and a zero
// exponent with one is the subnormal 2^-127; so one v_lshl_or_b32 serves every byte.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float((byte << 23) | 0x00400000u); }

// Two e2m1 values (byte S of w) times 2^(scale) in XT: exact in bf16; in fp16 exact for
// scales 2^-23 .. 2^13 and rounded once (or infinite) outside.
template <int XT, int S>
__device__ __forceinline__ uint32_t mx_weights2(uint32_t w, float scale) {
    if constexpr (XT == DT_BF16) return bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, S));
    else return bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, S));
}
template <int XT>
__device__ __forceinline__ uint4_t mx_weights8(uint32_t w, float scale) {
    uint4_t r;
    r[0] = mx_weights2<XT, 0>(w, scale);
    r[1] = mx_weights2<XT, 1>(w, scale);
    r[2] = mx_weights2<XT, 2>(w, scale);
    r[3] = mx_weights2<XT, 3>(w, scale);
    return r;
}

template <int XT>
__device__ __forceinline__ float4_t mx_mfma16(uint4_t a, uint4_t b, float4_t c) {
    if constexpr (XT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8_t>(a), bitcast<bf16x8_t>(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<half8_t>(a), bitcast<half8_t>(b), c, 0, 0, 0);
}

__device__ __forceinline__ int8v_t mx_operand(uint4_t v) {
    int8v_t r = {(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};   // e2m1: the first four registers
    return r;
}

// 128 K elements: lane l holds row l % 16, block l / 16 of either operand and that block's scale byte.
__device__ __forceinline__ float4_t mx_mfma16_fp4(uint4_t a, uint4_t b, float4_t c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(a), mx_operand(b), c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// Eight fp32 values as three bf16 pieces of 8 significant bits, each the upper half of what the
// ones before it left (cutting off, not rounding: the largest finite values stay finite).  An
// infinity or NaN is its first piece alone.
__device__ __forceinline__ void mx_split8(const float *x, uint4_t (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[2] = {x[2 * i], x[2 * i + 1]};
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            uint32_t h[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                h[e] = __float_as_uint(v[e]) & 0xFFFF0000u;
                const float rest = v[e] - __uint_as_float(h[e]);
                v[e] = s > 0 || (h[e] & 0x7F800000u) != 0x7F800000u ? rest : 0.f;
            }
            p[s][i] = (h[0] >> 16) | h[1];
        }
    }
}

// One fp32 value to the output type DT.
template <int DT>
__device__ __forceinline__ void mx_store(void *p, int64_t i, float v) {
    if constexpr (DT == DT_F32) ((float *)p)[i] = v;
    else if constexpr (DT == DT_BF16) ((__bf16 *)p)[i] = (__bf16)v;
    else ((_Float16 *)p)[i] = (_Float16)v;
}

template <int DT>
struct mx_type { typedef _Float16 T; };
template <>
struct mx_type<DT_BF16> { typedef __bf16 T; };
template <>
struct mx_type<DT_F32> { typedef float T; };

// Launchers (one per file), called by mcq4_mx_capi.cpp after its checks.
hipError_t launch_mx_quantize(const void *X, int x_dt, int64_t row_stride, int64_t col_stride, int64_t R, int64_t K,
                              uint8_t *packed, uint8_t *scales, hipStream_t s);
hipError_t launch_mx_dequantize(const uint8_t *packed, const uint8_t *scales, int64_t R, int64_t K, void *out, int out_dt,
                                hipStream_t s);
struct MxCall {
    const void *X;                 // [M][ldx] activations, or their packed e2m1 [M][K/2]
    const uint8_t *Xs;             // scale bytes [M][K/32] of microscaled activations, else null
    int x_dt;                      // type of X; of Y where X is microscaled
    int64_t ldx;
    const uint8_t *W, *Ws;         // packed [N][K/2], scales [N][K/32]
    void *Y;
    int64_t ldy, M, K, N;
};
hipError_t launch_mx_direct(const MxCall &c, hipStream_t s);
// Which kernel a product takes (mx_gemm.h, mx_plan.cpp), and the bytes that it needs behind the counter area.
struct MxPlan {
    int kind;
    int S;             // K splits
    size_t bytes;
};
MxPlan mx_plan(const MxCall &c);
size_t mx_workspace_bytes(const MxPlan &p);     // the counter area included, or 0
hipError_t launch_mx(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s);

}  // namespace mcq4
