// Shared parts of the LDS-staged MXFP4 products (mx_gemm.hip, mx_gemm4.hip): tile order,
// copies to LDS, the store of a tile and the sum of K splits.
#pragma once

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
// Adds S partials [S][M][ldp] in order and stores them in type dt (mx_gemm.hip).
hipError_t launch_mx_sum(const float *part, int S, void *Y, int64_t ldy, int dt, int64_t M, int64_t N, hipStream_t s);

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
