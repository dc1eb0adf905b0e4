// Writing to and reading from the 8-bit key/value cache (layout: kv8_common.h).
//
// Append: a page's scale for a head is the smallest power of two (2^-126 at least) that brings
// the largest finite magnitude of its new tokens to 448 or less, and no smaller than what the
// page has where it holds older tokens; those are then rescaled to it, which rounds only what
// falls into e4m3's subnormals.  Infinities and NaN become NaN.  A power of two makes the
// division exact, so a code carries e4m3's rounding alone.
//
// A workgroup takes a page's head.  Short kernels: 5121 tokens x 8 heads x 128 bf16 are appended in
// 10.8 us and read in 7.4 (31 MB each, 3.7 us at a copy's rate in the last-level cache), a token for
// each of 64 sequences in 7: a launch (2.5 us), the chain of lens, table, elements, scale, and the
// VALU, which was half of the time with elements and bytes taken one by one (14.8 and 9.6 us).
#include "kv8_common.h"

namespace mcq4 {

// fp32 values of 8 neighbouring elements.
template <int DT, bool VEC>
__device__ __forceinline__ void kv8_load8(const void *p, int64_t at, float (&x)[8]) {
    if constexpr (DT == DT_F32) {
        if constexpr (VEC) {
            const float4_t *q = (const float4_t *)((const float *)p + at);
            const float4_t u = q[0], v = q[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = u[i]; x[4 + i] = v[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = ((const float *)p)[at + i];
        }
    } else if constexpr (VEC) {
        const uint4_t u = *(const uint4_t *)((const uint16_t *)p + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t h = (uint16_t)(i & 1 ? u[i / 2] >> 16 : u[i / 2]);
            x[i] = DT == DT_BF16 ? __uint_as_float((uint32_t)h << 16) : (float)bitcast<_Float16>(h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t h = ((const uint16_t *)p)[at + i];
            x[i] = DT == DT_BF16 ? __uint_as_float((uint32_t)h << 16) : (float)bitcast<_Float16>(h);
        }
    }
}

__device__ __forceinline__ uint32_t kv8_codes4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Four codes times 2^-k, rounded again.
__device__ __forceinline__ uint32_t kv8_rescale4(uint32_t w, float f) {
    const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return kv8_codes4(a[0] * f, a[1] * f, b[0] * f, b[1] * f);
}
// 2^e of a whole number, 0 below the smallest normal one.
__device__ __forceinline__ float kv8_pow2(int e) { return e < -126 ? 0.f : __uint_as_float((uint32_t)(e + 127) << 23); }

// Bytes turned: a[i]'s byte j becomes byte i of the result's j.
__device__ __forceinline__ uint4_t kv8_turn4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    const uint32_t l0 = __builtin_amdgcn_perm(a1, a0, 0x05010400u), h0 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);
    const uint32_t l1 = __builtin_amdgcn_perm(a3, a2, 0x05010400u), h1 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
    return uint4_t{__builtin_amdgcn_perm(l1, l0, 0x05040100u), __builtin_amdgcn_perm(l1, l0, 0x07060302u),
                   __builtin_amdgcn_perm(h1, h0, 0x05040100u), __builtin_amdgcn_perm(h1, h0, 0x07060302u)};
}
// u / d for u < 2^16 by a multiplication with kv8_over(d), 1 < d <= 32.
__device__ __forceinline__ uint32_t kv8_over(int d) { return 0xFFFFFFFFu / (uint32_t)d + 1; }

// Codes of 8 neighbouring elements over 2^(byte - 127).  16-bit elements that are finite take the scaled conversion,
// which rounds the same way.
template <int DT, bool VEC>
__device__ __forceinline__ uint2_t kv8_encode8(const void *p, int64_t at, int byte, bool finite) {
    typedef short short2_t __attribute__((ext_vector_type(2)));
    if constexpr (DT != DT_F32 && VEC) {
        if (finite) {
            const uint4_t u = *(const uint4_t *)((const uint16_t *)p + at);
            const float s = __uint_as_float((uint32_t)byte << 23);
            short2_t r[2] = {{0, 0}, {0, 0}};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == DT_BF16) {
                    typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
                    r[i / 2] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r[i / 2], bitcast<bf2_t>(u[i]), s, true)
                                     : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r[i / 2], bitcast<bf2_t>(u[i]), s, false);
                } else {
                    r[i / 2] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r[i / 2], bitcast<half2_t>(u[i]), s, true)
                                     : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r[i / 2], bitcast<half2_t>(u[i]), s, false);
                }
            }
            return uint2_t{bitcast<uint32_t>(r[0]), bitcast<uint32_t>(r[1])};
        }
    }
    float f[8];
    kv8_load8<DT, VEC>(p, at, f);
    const float inv = kv8_pow2(127 - byte);
    return uint2_t{kv8_codes4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), kv8_codes4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv)};
}

__device__ __forceinline__ int kv8_touched(const Kv8Batch &t, int page_log, int b) {
    const int n = kv8_span(t, b).n, s = t.lens[b];
    return n > 0 && s >= 0 && s <= 0x7FFFFFFF - n ? ((s + n - 1) >> page_log) - (s >> page_log) + 1 : 0;
}

// A workgroup writes what a page's head gets of the keys (blockIdx.z 0) or the values (1).
constexpr int KVA_PITCH = 64 + 4;      // of a channel's 64 slots in LDS: rows of channels fall into different banks
template <int DT, bool VEC>
__global__ void __launch_bounds__(256)
kv8_append_kernel(Kv8Cache c, Kv8Batch t, Kv8Tokens kt, Kv8Tokens vt, int per_seq) {
    __shared__ uint32_t wave_max[4];
    __shared__ __attribute__((aligned(16))) uint8_t turn[256 * KVA_PITCH];
    const int tid = threadIdx.x, page = c.page(), h = blockIdx.y;
    const bool is_v = blockIdx.z;
    Kv8Item it;
    if (per_seq) it = {(int)blockIdx.x / per_seq, (int)blockIdx.x % per_seq};
    else it = kv8_locate((int)blockIdx.x, t.B, [&](int b) { return kv8_touched(t, c.page_log, b); });
    if (it.b >= t.B || it.i >= kv8_touched(t, c.page_log, it.b)) return;
    const Kv8Span sp = kv8_span(t, it.b);
    const int start = t.lens[it.b];
    const int p0 = ((start >> c.page_log) + it.i) << c.page_log;          // the page's first token
    const int id = kv8_page(t, c.P, c.page_log, it.b, p0);
    if (id < 0) return;
    const int lo = max(start, p0), nt = min(start + sp.n - lo, page - (lo - p0));      // p0 + page may be 2^31
    const Kv8Tokens x = is_v ? vt : kt;
    const int64_t x0 = (int64_t)(sp.first + lo - start) * x.token + (int64_t)h * x.head;
    const int D8 = c.D >> 3, units = nt * D8;

    uint8_t *scale = (is_v ? c.vs : c.ks) + (int64_t)id * c.H + h;
    const int was = lo > p0 ? *scale : 0;                // of the page's older tokens, if it has any

    const uint32_t over = kv8_over(D8);
    auto place = [&](int u) {                            // of 8 elements
        const int token = (int)__umulhi((uint32_t)u, over);
        return x0 + (int64_t)token * x.token + (u - token * D8) * 8;
    };
    auto largest = [&](uint32_t v) {                     // of all threads
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
        if ((tid & 63) == 0) wave_max[tid >> 6] = v;
        __syncthreads();
        return max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
    };
    // The largest finite magnitude, as fp32 bits.  16-bit elements: two at a time, and again one by one only where
    // one of them is not finite.
    uint32_t m = 0;
    bool finite = false;
    if constexpr (DT != DT_F32 && VEC) {
        typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
        ushort2_t pair = {0, 0};
        for (int u0 = 0; u0 < units; u0 += 4 * 256) {
            uint4_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w[k] = uint4_t{0, 0, 0, 0};
                if (u0 + 256 * k < units) w[k] = *(const uint4_t *)((const uint16_t *)x.p + place(min(u0 + 256 * k + tid, units - 1)));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) pair = __builtin_elementwise_max(pair, bitcast<ushort2_t>(w[k][i] & 0x7FFF7FFFu));
        }
        m = largest(max((uint32_t)pair[0], (uint32_t)pair[1]));
        finite = m < (DT == DT_BF16 ? 0x7F80u : 0x7C00u);
        m = DT == DT_BF16 ? m << 16 : __float_as_uint((float)bitcast<_Float16>((uint16_t)m));
    }
    if (!finite) {
        m = 0;
        for (int u = tid; u < units; u += 256) {
            float f[8];
            kv8_load8<DT, VEC>(x.p, place(u), f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = __float_as_uint(f[i]) & 0x7FFFFFFFu;
                if (b < 0x7F800000u && b > m) m = b;
            }
        }
        __syncthreads();                                 // wave_max has been read
        m = largest(m);
    }
    int byte = max((int)(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0), 1);

    uint8_t *codes = (is_v ? c.v : c.k) + ((int64_t)id * c.H + h) * page * c.D;
    const int older = lo - p0;
    if (older) {
        if (was >= byte) {
            byte = was;
        } else {
            const float f = kv8_pow2(was - byte);
            uint32_t *w = (uint32_t *)codes;
            if (!is_v) {
                for (int i = tid; i < older * c.D / 4; i += 256) w[i] = kv8_rescale4(w[i], f);
            } else {                                     // every channel's first `older` slots, the last word in part
                const int words = (older + 3) >> 2;
                for (int i = tid; i < c.D * words; i += 256) {
                    const int at = (i / words) * (page >> 2) + i % words, keep = older - 4 * (i % words);
                    const uint32_t v = w[at], r = kv8_rescale4(v, f), mask = keep >= 4 ? ~0u : (1u << (8 * keep)) - 1;
                    w[at] = (r & mask) | (v & ~mask);
                }
            }
        }
        __syncthreads();                                 // the new codes share words with the rescaled ones; `was` is read
    }
    if (tid == 0) *scale = (uint8_t)byte;
    if (!is_v) {
        uint2_t *dst = (uint2_t *)(codes + (int64_t)older * c.D);
#pragma unroll 4
        for (int u = tid; u < units; u += 256) dst[u] = kv8_encode8<DT, VEC>(x.p, place(u), byte, finite);
        return;
    }
    // Values: 64 slots of every channel at a time, turned in LDS.  A thread turns 4 slots (a dword) of 8 channels.
    const int slots = min(page, 64), words_log = slots == 64 ? 4 : slots == 32 ? 3 : 2;
    for (int s0 = older & ~63; s0 < older + nt; s0 += 64) {
        const int from = max(older, s0), to = min(older + nt, s0 + 64), w0 = (from - s0) >> 2, w1 = (to - s0 + 3) >> 2;
        for (int u = tid; u < (w1 - w0) * D8; u += 256) {
            const int n = (int)__umulhi((uint32_t)u, over), w = w0 + n, d = (u - n * D8) * 8;
            uint2_t r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {                // slots that are not of these tokens: some codes, not written below
                const int slot = min(max(s0 + 4 * w + e, from), to - 1);
                r[e] = kv8_encode8<DT, VEC>(x.p, x0 + (int64_t)(slot - older) * x.token + d, byte, finite);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4_t t = kv8_turn4(r[0][i], r[1][i], r[2][i], r[3][i]);
#pragma unroll
                for (int k = 0; k < 4; ++k) *(uint32_t *)(turn + (d + 4 * i + k) * KVA_PITCH + 4 * w) = t[k];
            }
        }
        __syncthreads();
        if (to - from == slots) {                        // whole: 16 bytes at a time
            for (int i = tid; i < c.D << (words_log - 2); i += 256) {
                const int d = i >> (words_log - 2), w = (i & ((1 << (words_log - 2)) - 1)) * 4;
                const uint32_t *src = (const uint32_t *)(turn + d * KVA_PITCH) + w;
                *(uint4_t *)(codes + d * page + s0 + 4 * w) = uint4_t{src[0], src[1], src[2], src[3]};
            }
        } else {
            for (int i = tid; i < c.D << words_log; i += 256) {
                const int d = i >> words_log, s = 4 * (i & ((1 << words_log) - 1));
                if (s0 + s + 4 <= from || s0 + s >= to) continue;
                uint8_t *dst = codes + d * page + s0 + s;
                const uint8_t *src = turn + d * KVA_PITCH + s;
                if (s0 + s >= from && s0 + s + 4 <= to) {
                    *(uint32_t *)dst = *(const uint32_t *)src;
                } else {
                    for (int e = 0; e < 4; ++e)
                        if (s0 + s + e >= from && s0 + s + e < to) dst[e] = src[e];
                }
            }
        }
        __syncthreads();
    }
}

// The values of a page's head, to [B][W page][H][D]; zero from the context's end on.
template <int DT>
__global__ void __launch_bounds__(256)
kv8_read_kernel(Kv8Cache c, Kv8Batch t, void *ko, void *vo) {
    __shared__ __attribute__((aligned(16))) uint8_t turn[64 * (256 + 8)];
    typedef typename mx_type<DT>::T T;
    const int tid = threadIdx.x, page = c.page(), h = blockIdx.y;
    const bool is_v = blockIdx.z;
    const int b = (int)(blockIdx.x / t.W), j = (int)(blockIdx.x % t.W);
    const int p0 = j << c.page_log, have = min(max(t.lens[b] - p0, 0), page);
    const int id = have ? kv8_page(t, c.P, c.page_log, b, p0) : -1;
    const int n = id < 0 ? 0 : have;
    const int64_t o = (((int64_t)b * t.W * page + p0) * c.H + h) * c.D;
    T *out = (T *)(is_v ? vo : ko) + o;
    const int64_t block = ((int64_t)max(id, 0) * c.H + h);
    const uint8_t *codes = (is_v ? c.v : c.k) + block * page * c.D;
    const float s = mx_scale((is_v ? c.vs : c.ks)[block]);
    // In fp32, whose multiplication takes the mantissa too: 2^-127 for byte 0, NaN for 255 (mx_common.h).
    const uint32_t bits = __float_as_uint(s);
    const float f = __uint_as_float(bits < 0x00800000u || bits > 0x7F800000u ? bits : bits & 0xFF800000u);
    const int D8 = c.D >> 3, slots = min(page, 64), words_log = slots == 64 ? 4 : slots == 32 ? 3 : 2;
    const uint32_t over = kv8_over(D8);
    for (int s0 = 0; s0 < page; s0 += 64) {
        if (is_v && s0 < n) {                            // a thread turns 4 slots (a dword) of 4 channels
            for (int i = tid; i < (c.D >> 2) << words_log; i += 256) {
                const int d = 4 * (i >> words_log), at = 4 * (i & ((1 << words_log) - 1));
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = *(const uint32_t *)(codes + (d + e) * page + s0 + at);
                const uint4_t t = kv8_turn4(w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) *(uint32_t *)(turn + (at + e) * (c.D + 8) + d) = t[e];
            }
        }
        __syncthreads();
#pragma unroll 2
        for (int u = tid; u < slots * D8; u += 256) {
            const int slot = (int)__umulhi((uint32_t)u, over), d = (u - slot * D8) * 8;
            T *dst = out + (int64_t)(s0 + slot) * c.H * c.D + d;
            uint2_t w = {0, 0};
            if (s0 + slot < n) w = is_v ? *(const uint2_t *)(turn + slot * (c.D + 8) + d) : *(const uint2_t *)(codes + (s0 + slot) * c.D + d);
            if constexpr (DT == DT_F32) {
                float4_t r[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2_t x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), y = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
                    r[i] = float4_t{x[0], x[1], y[0], y[1]};
                    if (s0 + slot < n) r[i] *= f;
                }
                ((float4_t *)dst)[0] = r[0];
                ((float4_t *)dst)[1] = r[1];
            } else {
                uint4_t r;
                const float sc = s0 + slot < n ? s : 1.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (DT == DT_BF16) {
                        r[2 * i] = bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], sc, false));
                        r[2 * i + 1] = bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], sc, true));
                    } else {
                        r[2 * i] = bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], sc, false));
                        r[2 * i + 1] = bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], sc, true));
                    }
                }
                *(uint4_t *)dst = r;
            }
        }
        __syncthreads();
    }
}

template <int DT>
static hipError_t launch_kv8_append_t(const Kv8Cache &c, const Kv8Batch &b, const Kv8Tokens &k, const Kv8Tokens &v, hipStream_t s) {
    // Touched pages: without offsets at most per_seq for each sequence; with them, over all sequences, a page for
    // every whole page of tokens and two for the ends.
    const int per_seq = b.cu ? 0 : (b.each + c.page() - 2) / c.page() + 1;
    const int64_t items = b.cu ? (int64_t)b.T / c.page() + 2 * (int64_t)b.B : (int64_t)b.B * per_seq;
    constexpr int e16 = DT == DT_F32 ? 4 : 8;
    bool vec = true;
    for (const Kv8Tokens *x : {&k, &v}) vec = vec && (uintptr_t)x->p % 16 == 0 && x->token % e16 == 0 && x->head % e16 == 0;
    const dim3 grid((unsigned)items, (unsigned)c.H, 2);
    if (vec) hipLaunchKernelGGL((kv8_append_kernel<DT, true>), grid, dim3(256), 0, s, c, b, k, v, per_seq);
    else hipLaunchKernelGGL((kv8_append_kernel<DT, false>), grid, dim3(256), 0, s, c, b, k, v, per_seq);
    return hipGetLastError();
}

hipError_t launch_kv8_append(const Kv8Cache &c, const Kv8Batch &b, const Kv8Tokens &k, const Kv8Tokens &v, int dt, hipStream_t s) {
    if (dt == DT_F16) return launch_kv8_append_t<DT_F16>(c, b, k, v, s);
    if (dt == DT_BF16) return launch_kv8_append_t<DT_BF16>(c, b, k, v, s);
    return launch_kv8_append_t<DT_F32>(c, b, k, v, s);
}

hipError_t launch_kv8_read(const Kv8Cache &c, const Kv8Batch &b, void *k, void *v, int dt, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)b.B * b.W), (unsigned)c.H, 2);
    if (dt == DT_F16) hipLaunchKernelGGL(kv8_read_kernel<DT_F16>, grid, dim3(256), 0, s, c, b, k, v);
    else if (dt == DT_BF16) hipLaunchKernelGGL(kv8_read_kernel<DT_BF16>, grid, dim3(256), 0, s, c, b, k, v);
    else hipLaunchKernelGGL(kv8_read_kernel<DT_F32>, grid, dim3(256), 0, s, c, b, k, v);
    return hipGetLastError();
}

}  // namespace mcq4
