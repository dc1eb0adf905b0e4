// MXFP4 conversions (format: mx_common.h).
//
// Quantize, OCP MX v1.0 section 6.3: a block's scale is 2^(floor(log2(amax)) - 2), 2 being
// e2m1's largest exponent, an element x / scale rounded to nearest even and saturated at 6.
// The exponent is read off the bits of amax, and the division by a power of two is exact, so
// the one rounding is e2m1's own; v_cvt_scalef32_pk_fp4_f32 does both.  A block that holds an
// infinity or a NaN has no scale: its byte is 255 (NaN) and its elements are 0.
//
// Bound by memory: 14336 x 4096 bf16 is quantized in 25.6 us (5.8 TB/s read and written) and
// dequantized in 22.3 (6.6 TB/s), where a copy reaches 4.9 TB/s from memory and 8.5 out of the
// last-level cache.  1001 x 4096 fp32 held [K, N] is quantized in 6.7 us (2.8 TB/s: a wave's 256
// bytes of a row are not aligned, and 256 workgroups have one turn each), dequantized in 4.2.
#include "mx_common.h"

namespace mcq4 {

constexpr int MXQ_U = 4;   // pieces of 8 elements per thread, their loads in flight together

// fp32 bits of 8 consecutive elements.
template <int DT, bool VEC>
__device__ __forceinline__ void mx_load8(const void *X, int64_t at, uint32_t (&b)[8]) {
    if constexpr (DT == DT_F32) {
        if constexpr (VEC) {
            const uint4_t *p = (const uint4_t *)((const float *)X + at);
            const uint4_t u = p[0], v = p[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) { b[i] = u[i]; b[4 + i] = v[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = ((const uint32_t *)X)[at + i];
        }
    } else {
        uint32_t h[8];
        if constexpr (VEC) {
            const uint4_t u = *(const uint4_t *)((const uint16_t *)X + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = i & 1 ? u[i / 2] >> 16 : u[i / 2] & 0xFFFFu;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = ((const uint16_t *)X)[at + i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            b[i] = DT == DT_BF16 ? h[i] << 16 : __float_as_uint((float)bitcast<_Float16>((uint16_t)h[i]));
    }
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// Largest magnitude as bits: infinities and NaN are above every finite value.
__device__ __forceinline__ uint32_t mx_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
__device__ __forceinline__ uint32_t mx_codes8(const uint32_t *b, uint32_t byte) {
    if (byte == 255) return 0;
    const float s = mx_scale(byte);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(b[0]), __uint_as_float(b[1]), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(b[2]), __uint_as_float(b[3]), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(b[4]), __uint_as_float(b[5]), s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __uint_as_float(b[6]), __uint_as_float(b[7]), s, 3);
}

// Rows whose elements are neighbours: four lanes to a block, 8 elements each, so a wave reads
// 1 or 2 KiB and writes 256 bytes of codes in one piece.  FLAT: the rows follow each other.
template <int DT, bool VEC, bool FLAT>
__global__ void __launch_bounds__(256)
mx_quantize_rows_kernel(const void *__restrict__ X, int64_t row_stride, uint32_t units, uint32_t row_units,
                        uint8_t *__restrict__ packed, uint8_t *__restrict__ scales) {
    const uint32_t u0 = blockIdx.x * (256 * MXQ_U) + threadIdx.x;
    uint32_t b[MXQ_U][8];
#pragma unroll
    for (int i = 0; i < MXQ_U; ++i) {
        const uint32_t u = min(u0 + 256 * i, units - 1);      // a whole block's lanes are clamped together or not at all
        const int64_t at = FLAT ? (int64_t)u * 8 : (int64_t)(u / row_units) * row_stride + (int64_t)(u % row_units) * 8;
        mx_load8<DT, VEC>(X, at, b[i]);
    }
#pragma unroll
    for (int i = 0; i < MXQ_U; ++i) {
        const uint32_t u = u0 + 256 * i;
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = umax(m, b[i][j] & 0x7FFFFFFFu);
        m = umax(m, __builtin_amdgcn_update_dpp(0, m, 0xB1, 0xF, 0xF, true));   // lanes 1 0 3 2
        m = umax(m, __builtin_amdgcn_update_dpp(0, m, 0x4E, 0xF, 0xF, true));   // lanes 2 3 0 1
        const uint32_t byte = mx_byte(m), w = mx_codes8(b[i], byte);
        if (u < units) {
            ((uint32_t *)packed)[u] = w;
            if ((u & 3) == 0) scales[u >> 2] = (uint8_t)byte;
        }
    }
}

// Any strides, meant for a matrix held [K, R] and passed as its transpose: a lane owns a row
// and reads 32 elements that lie a column stride apart, so a wave reads 64 neighbours at a
// time.  A workgroup's 64 rows x 8 blocks go through LDS, from which each row's 128 bytes of
// codes are written in one piece.
constexpr int MXQ_PITCH = 8 * 16 + 16;
template <int DT>
__global__ void __launch_bounds__(256)
mx_quantize_cols_kernel(const void *__restrict__ X, int64_t row_stride, int64_t col_stride, int64_t R, int64_t nb,
                        uint8_t *__restrict__ packed, uint8_t *__restrict__ scales) {
    __shared__ __attribute__((aligned(16))) uint8_t codes[64 * MXQ_PITCH];
    __shared__ uint8_t bytes[64 * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r0 = (int64_t)blockIdx.x * 64, kb0 = (int64_t)blockIdx.y * 8;
    const int64_t r = r0 + lane < R ? r0 + lane : R - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int k = 2 * wave + i;
        if (kb0 + k < nb) {
            const int64_t at = r * row_stride + (kb0 + k) * MX_BLOCK * col_stride;
            uint32_t b[MX_BLOCK], m = 0;
#pragma unroll
            for (int j = 0; j < MX_BLOCK; ++j) {
                if constexpr (DT == DT_F32) b[j] = ((const uint32_t *)X)[at + j * col_stride];
                else if constexpr (DT == DT_BF16) b[j] = (uint32_t)((const uint16_t *)X)[at + j * col_stride] << 16;
                else b[j] = __float_as_uint((float)((const _Float16 *)X)[at + j * col_stride]);
            }
#pragma unroll
            for (int j = 0; j < MX_BLOCK; ++j) m = umax(m, b[j] & 0x7FFFFFFFu);
            const uint32_t byte = mx_byte(m);
            uint4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = mx_codes8(b + 8 * j, byte);
            *(uint4_t *)(codes + lane * MXQ_PITCH + 16 * k) = w;
            bytes[lane * 8 + k] = (uint8_t)byte;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = threadIdx.x + 256 * i, row = t >> 3, k = t & 7;
        if (r0 + row < R && kb0 + k < nb) {
            const int64_t block = (r0 + row) * nb + kb0 + k;
            *(uint4_t *)(packed + block * 16) = *(const uint4_t *)(codes + row * MXQ_PITCH + 16 * k);
            scales[block] = bytes[row * 8 + k];
        }
    }
}

// A lane turns 4 bytes of codes into 8 values: a wave reads 256 bytes and writes 1 or 2 KiB
// in one piece.  The values are exact in fp32 and bf16 and rounded once in fp16 (mx_common.h).
template <int DT>
__global__ void __launch_bounds__(256)
mx_dequantize_kernel(const uint8_t *__restrict__ packed, const uint8_t *__restrict__ scales, uint32_t units,
                     void *__restrict__ out) {
    const uint32_t u0 = blockIdx.x * (256 * MXQ_U) + threadIdx.x;
    uint32_t w[MXQ_U], byte[MXQ_U];
#pragma unroll
    for (int i = 0; i < MXQ_U; ++i) {
        const uint32_t u = min(u0 + 256 * i, units - 1);
        w[i] = ((const uint32_t *)packed)[u];
        byte[i] = scales[u >> 2];
    }
#pragma unroll
    for (int i = 0; i < MXQ_U; ++i) {
        const uint32_t u = u0 + 256 * i;
        if (u >= units) return;
        const float s = mx_scale(byte[i]);
        if constexpr (DT == DT_F32) {
            float2_t v[4];
            v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 0);
            v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 1);
            v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 2);
            v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 3);
            float4_t *p = (float4_t *)((float *)out + (int64_t)u * 8);
            p[0] = float4_t{v[0][0], v[0][1], v[1][0], v[1][1]};
            p[1] = float4_t{v[2][0], v[2][1], v[3][0], v[3][1]};
        } else {
            *(uint4_t *)((uint16_t *)out + (int64_t)u * 8) = mx_weights8<DT>(w[i], s);
        }
    }
}

template <int DT>
static hipError_t launch_mx_quantize_t(const void *X, int64_t rs, int64_t cs, int64_t R, int64_t K, uint8_t *packed,
                                       uint8_t *scales, hipStream_t s) {
    const int es = DT == DT_F32 ? 4 : 2;
    if (cs != 1) {
        hipLaunchKernelGGL(mx_quantize_cols_kernel<DT>, dim3((unsigned)((R + 63) / 64), (unsigned)((K / MX_BLOCK + 7) / 8)),
                           dim3(256), 0, s, X, rs, cs, R, K / MX_BLOCK, packed, scales);
        return hipGetLastError();
    }
    const bool flat = rs == K, vec = (uintptr_t)X % 16 == 0 && rs * es % 16 == 0;
    const uint32_t row_units = (uint32_t)(K / 8), units = (uint32_t)(R * (K / 8));
    const dim3 grid((unsigned)(((int64_t)units + 256 * MXQ_U - 1) / (256 * MXQ_U))), block(256);
    if (vec && flat) hipLaunchKernelGGL((mx_quantize_rows_kernel<DT, true, true>), grid, block, 0, s, X, rs, units, row_units, packed, scales);
    else if (vec) hipLaunchKernelGGL((mx_quantize_rows_kernel<DT, true, false>), grid, block, 0, s, X, rs, units, row_units, packed, scales);
    else hipLaunchKernelGGL((mx_quantize_rows_kernel<DT, false, false>), grid, block, 0, s, X, rs, units, row_units, packed, scales);
    return hipGetLastError();
}

hipError_t launch_mx_quantize(const void *X, int x_dt, int64_t row_stride, int64_t col_stride, int64_t R, int64_t K,
                              uint8_t *packed, uint8_t *scales, hipStream_t s) {
    if (x_dt == DT_F16) return launch_mx_quantize_t<DT_F16>(X, row_stride, col_stride, R, K, packed, scales, s);
    if (x_dt == DT_BF16) return launch_mx_quantize_t<DT_BF16>(X, row_stride, col_stride, R, K, packed, scales, s);
    return launch_mx_quantize_t<DT_F32>(X, row_stride, col_stride, R, K, packed, scales, s);
}

hipError_t launch_mx_dequantize(const uint8_t *packed, const uint8_t *scales, int64_t R, int64_t K, void *out, int out_dt,
                                hipStream_t s) {
    const uint32_t units = (uint32_t)(R * (K / 8));
    const dim3 grid((unsigned)(((int64_t)units + 256 * MXQ_U - 1) / (256 * MXQ_U))), block(256);
    if (out_dt == DT_F16) hipLaunchKernelGGL(mx_dequantize_kernel<DT_F16>, grid, block, 0, s, packed, scales, units, out);
    else if (out_dt == DT_BF16) hipLaunchKernelGGL(mx_dequantize_kernel<DT_BF16>, grid, block, 0, s, packed, scales, units, out);
    else hipLaunchKernelGGL(mx_dequantize_kernel<DT_F32>, grid, block, 0, s, packed, scales, units, out);
    return hipGetLastError();
}

}  // namespace mcq4
