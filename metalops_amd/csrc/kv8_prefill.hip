// Attention over the 8-bit cache, many rows: tiles of 256 (D > 128: 128) query rows of a key/value
// head (a row is a new token and one of the head's G queries, G neighbouring rows to a token).
//
// Eight waves (D > 128: four) with 32 rows each go through the context 64 tokens at a time.  The
// workgroup turns a piece of K and V into 16 bits once, on its way from memory through registers
// to LDS (the next piece's loads in flight during a piece's products; one barrier a piece).
// 32 rows a wave: with 64, K and V would be read from LDS half as often, but the accumulators
// and two halves' scores need more than 256 registers, and the moves to and from the second 256
// cost more than the reads.  256 rows a workgroup halve what is converted for each of them: two
// prompts (2048 tokens of 4096, 1500 of 1500; 32 heads, 8 of keys, D = 128, causal) took 185 us
// with 128 rows and take 151.
// Both products are v_mfma_f32_32x32x16 with the cache as the A operand, so a lane's results
// belong to one row (l % 32):
//   S^T = K q^T    two tiles of 32 tokens.  A lane holds rows 8 (r / 4) + 4 (l / 32) + r % 4 of a
//                  tile; K's tokens are dealt to the tile's rows so that registers 8 j .. 8 j + 7
//                  are tokens 16 j + 8 (l / 32) .. + 7, and P needs no move between lanes in
//   O^T += V^T P^T whose operand from LDS is 8 such tokens of a channel.
// K lies in LDS token by token, V channel by channel, in rows of an odd number of 16 bytes, so
// that 16 lanes reading 16 rows meet 16 banks.
//
// A piece is taken in halves of 32 tokens: the exponentials of one (VALU) run between the products
// of the next one's S (matrix cores), the next one's maxima and the conversion of the next piece
// between the products with V.  So K is a piece ahead of V in LDS, in three buffers (D > 192: two).
//
// Scales, rounding and what is masked are as in kv8_attend.hip: K's scale multiplies the scores
// in fp32, V's goes into P, which is fp16 (kv8_attend.h).  A row's m and k follow only once its scores
// exceed m by KVP_LAG, or P might exceed 2^15, so that most pieces leave the accumulators alone; P
// stands as high as that allows, and weights keep 11 bits down to 2^-21 of the largest one.
//
// Bound by the matrix cores and the VALU between their products: those prompts are 122 GFLOP,
// 0.80 PFLOP/s, where a library product of large fp16 matrices reaches 1.15 on this card.
#include <algorithm>
#include <atomic>

#include "kv8_prompt.h"

namespace mcq4 {

// NT: tiles of 32 channels.
template <int QT, int NT>
__global__ void __launch_bounds__(64 * kvp_waves(NT), 1)
kv8_prefill_kernel(Kv8Attend a, Kv8Plan p) {
    constexpr int WAVES = kvp_waves(NT), ROWS = KVP_WAVE_ROWS * WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    // Neighbouring workgroups take neighbouring heads: with 8 of them an XCD's L2 serves one.
    const int h = (int)(blockIdx.x % (uint32_t)a.cache.H), tile = (int)(blockIdx.x / (uint32_t)a.cache.H);
    if (a.batch.cu && blockIdx.y == 0) kv8_rest(a, blockIdx.x, gridDim.x);
    Kv8Rows R;
    if (!kv8_longest_first(a, tile, ROWS, R)) return;
    kv8_uniform(R);
    const int split = blockIdx.y, parts = kv8_parts(R, p);
    if (split >= parts) return;
    const int c0 = R.lo + split * p.span, c1 = split == parts - 1 ? R.hi : c0 + p.span;
    kvp_attend<QT, NT, WAVES, kvp_k_buffers(NT), kvp_ahead(NT)>(a, a.batch, a.causal, a.window, R, h, c0, c1, smem,
                                                 [&](int row, int end_hi, const float16_t (&acc)[NT], int unit, float m, float l) {
        const int D = a.cache.D, at_r = R.r0 + row;
        if (parts > 1 || a.pre.at) {
            const int64_t at = (((int64_t)tile * a.cache.H + h) * p.splits + split) * ROWS + row;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (32 * i + 8 * e < D)
                        *(float4_t *)(p.acc + at * D + 32 * i + 8 * e + 4 * end_hi) =
                            float4_t{__builtin_ldexpf(acc[i][4 * e], unit), __builtin_ldexpf(acc[i][4 * e + 1], unit),
                                     __builtin_ldexpf(acc[i][4 * e + 2], unit), __builtin_ldexpf(acc[i][4 * e + 3], unit)};
            if (end_hi == 0) *(float2_t *)(p.ml + at * 2) = float2_t{m, l};
            return;
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int64_t at_q = ((int64_t)(R.first_token + at_r / a.G) * a.cache.H + h) * a.G + at_r % a.G;      // token and head
        uint16_t *out = (uint16_t *)a.out + at_q * D + 4 * end_hi;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (32 * i + 8 * e < D) {
                    typedef typename mx_type<QT>::T T;
                    T v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = (T)__builtin_ldexpf(acc[i][4 * e + k] * inv, unit);
                    *(uint2_t *)(out + 32 * i + 8 * e) = bitcast<uint2_t>(v);
                }
        if (a.lse && end_hi == 0) a.lse[at_q] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * (1.0f / LOG2E);
    });
}

template <int QT, int NT>
static hipError_t launch_kv8_prefill_t(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    constexpr int lds = kvp_k_buffers(NT) * kvp_k_bytes(NT) + 2 * kvp_v_bytes(NT);
    static_assert(lds + 16 * kvp_channels(NT) + 64 <= 160 * 1024, "LDS budget");
    static std::atomic<uint64_t> done{0};
    if (lds > 64 * 1024)
        if (hipError_t e = mx_allow_lds((const void *)kv8_prefill_kernel<QT, NT>, lds, done)) return e;
    hipLaunchKernelGGL((kv8_prefill_kernel<QT, NT>), dim3((unsigned)p.tiles * (unsigned)a.cache.H, (unsigned)p.splits), dim3(64 * kvp_waves(NT)), lds, s, a, p);
    return hipGetLastError();
}

template <int QT>
static hipError_t launch_kv8_prefill_q(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    switch ((a.cache.D + 31) / 32) {
        case 1: return launch_kv8_prefill_t<QT, 1>(a, p, s);
        case 2: return launch_kv8_prefill_t<QT, 2>(a, p, s);
        case 3: return launch_kv8_prefill_t<QT, 3>(a, p, s);
        case 4: return launch_kv8_prefill_t<QT, 4>(a, p, s);
        case 5: return launch_kv8_prefill_t<QT, 5>(a, p, s);
        case 6: return launch_kv8_prefill_t<QT, 6>(a, p, s);
        case 7: return launch_kv8_prefill_t<QT, 7>(a, p, s);
        default: return launch_kv8_prefill_t<QT, 8>(a, p, s);
    }
}

hipError_t launch_kv8_prefill(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    return a.q_dt == DT_BF16 ? launch_kv8_prefill_q<DT_BF16>(a, p, s) : launch_kv8_prefill_q<DT_F16>(a, p, s);
}

}  // namespace mcq4
