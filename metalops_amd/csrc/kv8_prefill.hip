// Attention over the 8-bit cache, many rows: tiles of 128 query rows of a key/value head (a row
// is a new token and one of the head's G queries, G neighbouring rows to a token).
//
// Four waves with 32 rows each go through the context 64 tokens at a time.  The workgroup turns
// a piece of K and V into 16 bits once, on its way from memory through registers to LDS (two
// buffers, the next piece's loads in flight during a piece's products; one barrier a piece).
// Both products are v_mfma_f32_32x32x16 with the cache as the A operand, so a lane's results
// belong to one row (l % 32):
//   S^T = K q^T    two tiles of 32 tokens.  A lane holds rows 8 (r / 4) + 4 (l / 32) + r % 4 of a
//                  tile; K's tokens are dealt to the tile's rows so that registers 8 j .. 8 j + 7
//                  are tokens 16 j + 8 (l / 32) .. + 7, and P needs no move between lanes in
//   O^T += V^T P^T whose operand from LDS is 8 such tokens of a channel.
// K lies in LDS token by token, V channel by channel, in rows of an odd number of 16 bytes, so
// that 16 lanes reading 16 rows meet 16 banks.
//
// Scales, rounding and what is masked are as in kv8_attend.hip: K's scale multiplies the scores
// in fp32; V's is applied by the conversion, relative to the largest one met so far; P is fp16.
// The running maximum follows a row's scores once they exceed it by 2^8 (P stays far below
// fp16's 65504), so that most pieces leave the accumulators alone.
//
// 121 GFLOP of two bf16 prompts (2048 of 4096 and 1500 of 1500 tokens, 32 heads, D = 128).
#include <algorithm>
#include <atomic>

#include "kv8_attend.h"

namespace mcq4 {

constexpr int KVP_WAVES = 4;
static_assert(KVP_ROWS == 32 * KVP_WAVES, "32 rows a wave");
constexpr int KVP_V_PITCH = KVD_STEP * 2 + 16;
constexpr int kvp_pieces(int NT) { return (NT + 1) / 2; }            // 64 channels each
constexpr int kvp_k_pitch(int NT) { return 128 * kvp_pieces(NT) + 16; }
constexpr int kvp_buffer(int NT) { return KVD_STEP * kvp_k_pitch(NT) + 64 * kvp_pieces(NT) * KVP_V_PITCH; }

__device__ __forceinline__ float kvp_other(float x) {      // the value of lane l ^ 32
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? p[0] : p[1]);
}

template <int QT>
__device__ __forceinline__ float16_t kvp_mfma(uint4_t a, uint4_t b, float16_t c) { return mfma32<QT>(bitcast<half8_t>(a), bitcast<half8_t>(b), c); }

// 16 codes as 16-bit values times s, to 32 bytes of LDS.
template <int QT>
__device__ __forceinline__ void kvp_put(uint8_t *dst, uint4_t w, float s) {
    *(uint4_t *)dst = kv8_eight<QT>(w[0], w[1], s);
    *(uint4_t *)(dst + 16) = kv8_eight<QT>(w[2], w[3], s);
}

// NT: tiles of 32 channels.
template <int QT, int NT>
__global__ void __launch_bounds__(64 * KVP_WAVES, NT <= 4 ? 2 : 1)
kv8_prefill_kernel(Kv8Attend a, Kv8Plan p) {
    constexpr int NC = kvp_pieces(NT);
    constexpr int K_PITCH = kvp_k_pitch(NT), K_BYTES = KVD_STEP * K_PITCH, BUF = kvp_buffer(NT);
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ int nan_flag[2];
    __shared__ __attribute__((aligned(8))) uint16_t nan_map[2][64 * NC][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hi = lane >> 5;
    // Neighbouring workgroups take neighbouring heads: with 8 of them an XCD's L2 serves one.
    const int h = (int)(blockIdx.x % (uint32_t)a.cache.H), tile = (int)(blockIdx.x / (uint32_t)a.cache.H);
    Kv8Rows R;
    if (!kv8_longest_first(a, tile, KVP_ROWS, R)) return;
    kv8_uniform(R);
    const int split = blockIdx.y, parts = kv8_parts(R, p);
    if (split >= parts) return;
    const int c0 = R.lo + split * p.span, c1 = split == parts - 1 ? R.hi : c0 + p.span;

    const Kv8Cache &c = a.cache;
    const int D = c.D, page_log = c.page_log, page = 1 << page_log;
    // This lane's row, and what it and its wave's rows see.
    const int w0 = min(R.r0 + 32 * wave, R.rows - 1), w1 = min(R.r0 + 32 * wave + 31, R.rows - 1);
    const bool rows_here = R.r0 + 32 * wave < R.rows;
    const int r = min(R.r0 + 32 * wave + col, R.rows - 1);
    const int tok = r / a.G, head = h * a.G + r % a.G, pos = R.pos0 + tok;
    const int see_hi = a.causal ? min(pos + 1, R.ctx) : R.ctx, see_lo = a.window ? max(pos - a.window + 1, 0) : 0;
    const int pos_a = R.pos0 + w0 / a.G, pos_z = R.pos0 + w1 / a.G;
    const int all_hi = a.causal ? pos_a + 1 : R.ctx, all_lo = a.window ? pos_z - a.window + 1 : 0;
    const int any_hi = a.causal ? min(pos_z + 1, R.ctx) : R.ctx, any_lo = a.window ? pos_a - a.window + 1 : 0;

    // What all rows of the workgroup see (a page that is missing aside).
    const int tile_hi = a.causal ? min(R.pos0 + R.r0 / a.G + 1, R.ctx) : R.ctx;
    const int tile_lo = a.window ? R.pos0 + (min(R.r0 + KVP_ROWS, R.rows) - 1) / a.G - a.window + 1 : 0;

    const uint16_t *q = (const uint16_t *)a.q + (int64_t)(R.first_token + tok) * a.q_token + (int64_t)head * a.q_head;
    uint4_t qv[2 * NT];
#pragma unroll
    for (int k = 0; k < 2 * NT; ++k) qv[k] = 16 * k < D ? *(const uint4_t *)(q + 16 * k + 8 * hi) : uint4_t{0, 0, 0, 0};

    float16_t acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float qk = a.scale * LOG2E;

    // The thread's part of a piece: K token tid / 4 (a wave's 16 lie in one page), 16-byte pieces
    // tid % 4 + 4 i; V channels tid / 4 + 64 i, tokens 16 (tid % 4) ..  Channels past D repeat the
    // last ones: q is 0 there, and those of V are not stored.
    const int part = tid & 3, line = tid >> 2;
    uint4_t kr[NC], vr[NC];
    int ek, ev;                                          // table entries of the piece to be fetched
    auto pages = [&](int ci) {
        ek = kv8_entry(a.batch, page_log, R.b, ci * KVD_STEP + line);
        ev = kv8_entry(a.batch, page_log, R.b, ci * KVD_STEP + 16 * part);
    };
    // Scale bytes of tokens 16 (tid % 4) .., and whether the page is there.
    uint32_t kb_next = 0, vb_next = 0;
    bool there_next = false;
    int vref = 0, vref_next = 0;
    auto fetch = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        const int idk = kv8_checked(ek, c.P, t0 + (line & ~15), R.ctx), idv = kv8_checked(ev, c.P, t0 + 16 * part, R.ctx);
        const int64_t bk = (int64_t)max(idk, 0) * c.H + h, bv = (int64_t)max(idv, 0) * c.H + h;
        there_next = idv >= 0;
        kb_next = c.ks[bv];
        vb_next = c.vs[bv];
        const uint8_t *kp = c.k + (bk * page + ((t0 + line) & (page - 1))) * D;
        const uint8_t *vp = c.v + bv * page * D + ((t0 + 16 * part) & (page - 1));
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            kr[i] = *(const uint4_t *)(kp + min(16 * part + 64 * i, D - 16));
            vr[i] = *(const uint4_t *)(vp + min(line + 64 * i, D - 1) * page);
        }
    };
    // The fetched piece to buffer `buf`.
    auto put = [&](int buf, int piece) {
        uint8_t *kd = smem + buf * BUF + line * K_PITCH + 32 * part, *vd = smem + buf * BUF + K_BYTES + line * KVP_V_PITCH + 32 * part;
        const int mine = there_next ? (int)vb_next : 0;
        int top = max(mine, __shfl_xor(mine, 1));
        top = max(top, __shfl_xor(top, 2));
        vref_next = max(vref_next, __builtin_amdgcn_readfirstlane(top));
        const int rel = mine - vref_next;
        const float vs = rel < -100 ? 0x1p-100f : __uint_as_float((uint32_t)(rel + 127) << 23);
        if (!__all(there_next)) {                        // what page 0 holds there is not seen
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (!there_next) vr[i] = uint4_t{0, 0, 0, 0};
        }
        if (piece * KVD_STEP < tile_lo || (piece + 1) * KVD_STEP > tile_hi) {
            // Not every row sees every token: NaN of V would reach rows by 0 * NaN.  They become 0, and a map of them,
            // 64 tokens a channel, says which rows get one (NaN codes elsewhere are NaN by themselves).
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                uint32_t map = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t bad = ((vr[i][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                    vr[i][w] &= ~((bad >> 7) * 0xFFu);
                    map |= (((bad >> 7) * 0x10204080u) >> 28) << (4 * w);
                }
                nan_map[buf][line + 64 * i][part] = (uint16_t)map;
                if (map) nan_flag[buf] = piece + 1;
            }
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            kvp_put<QT>(kd + 128 * i, kr[i], 1.0f);
            kvp_put<DT_F16>(vd + 64 * i * KVP_V_PITCH, vr[i], vs);
        }
    };

    // K row of S-tile row l % 32: rows 16 j + 8 e + 4 h + i are tokens 16 j + 8 h + 4 e + i.
    const int k_row = (col & 16) | ((col & 4) << 1) | ((col & 8) >> 1) | (col & 3);
    const uint32_t lds0 = lds_addr(smem);
    const uint32_t k_off = lds0 + k_row * K_PITCH + 16 * hi, v_off = lds0 + K_BYTES + col * KVP_V_PITCH + 16 * hi;
    typedef __attribute__((address_space(3))) uint4_t lds_vec;
    auto lds16 = [&](uint32_t at) { return *(const lds_vec *)lds_ptr(at); };

    if (tid < 2) nan_flag[tid] = 0;                      // piece + 1 where a buffer's V has a NaN
    if (c0 < c1) {
        pages(c0);
        fetch(c0);
        pages(c0 + 1);
        __syncthreads();                                 // nan_flag
        put(0, c0);
    }
    wait_vmcnt<0>();                                     // q too: nothing in the loop waits for it again
    for (int ci = c0; ci < c1; ++ci) {
        const int buf = (ci - c0) & 1, t0 = ci * KVD_STEP;
        uint32_t kb[4];                                  // by groups of 16 tokens; bit 8: not there
#pragma unroll
        for (int g = 0; g < 4; ++g) kb[g] = (uint32_t)__builtin_amdgcn_readlane((int)(there_next ? kb_next : 256u), g);
        const int top = vref_next;
        if (ci + 1 < c1) {
            fetch(ci + 1);
            if (ci + 2 < c1) pages(ci + 2);
        }
        lds_barrier();                                   // the piece is in LDS, the other buffer has been read
        const bool has_nan = nan_flag[buf] == ci + 1;
        if (rows_here && t0 < any_hi && t0 + KVD_STEP > any_lo) {
            float16_t s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * NT; ++k)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    s[t] = kvp_mfma<QT>(lds16(k_off + buf * BUF + 32 * t * K_PITCH + 32 * k), qv[k], s[t]);
            const bool full = t0 >= all_lo && t0 + KVD_STEP <= all_hi && !((kb[0] | kb[1] | kb[2] | kb[3]) & 256u);
            uint32_t seen = ~0u;                         // bit 16 t + e: the row sees the token of s[t][e]
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float ks = qk * __uint_as_float((kb[2 * t + j] & 255u) << 23);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[t][8 * j + e] *= ks;
                }
            if (!full) {
                seen = 0;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int at = t0 + 16 * g + 8 * hi, from = min(max(see_lo - at, 0), 8), to = min(max(see_hi - at, 0), 8);
                    const uint32_t bits = kb[g] & 256u ? 0u : ((1u << to) - 1) & ~((1u << from) - 1);
                    seen |= bits << (8 * g);
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint32_t keep = (uint32_t)((int)(seen << (31 - 16 * t - e)) >> 31);
                        s[t][e] = __uint_as_float((__float_as_uint(s[t][e]) & keep) | (0xFF800000u & ~keep));
                    }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
            mx = fmaxf(mx, kvp_other(mx));
            const bool moved = mx > m + 8.f;             // also where m is -inf and mx is not
            if (__any(moved) || top > vref) {
                const float m_new = moved ? mx : m, m_use = m_new == -INFINITY ? 0.f : m_new;
                float shrink = __builtin_amdgcn_exp2f(m - m_use);
                m = m_new;
                l *= shrink;
                const int e = vref - top;
                shrink *= e < -126 ? 0.f : __uint_as_float((uint32_t)(e + 127) << 23);
                vref = top;
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i] *= shrink;
            }
            const float m_use = m == -INFINITY ? 0.f : m;
            uint4_t pr[2][2];
            float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = __builtin_amdgcn_exp2f(s[t][8 * j + 2 * e] - m_use), y = __builtin_amdgcn_exp2f(s[t][8 * j + 2 * e + 1] - m_use);
                        add[2 * t + j] += x + y;
                        pr[t][j][e] = bitcast<uint32_t>(half2_t{(_Float16)x, (_Float16)y});
                    }
            l += (add[0] + add[1]) + (add[2] + add[3]);
            const uint32_t vb0 = v_off + buf * BUF;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        acc[i] = kvp_mfma<DT_F16>(lds16(vb0 + 32 * i * KVP_V_PITCH + 64 * t + 32 * j), pr[t][j], acc[i]);
            if (has_nan) {
                // The row's tokens lie in two lanes, hi's eight of every 16; register r of acc[i] is channel 32 i + 8 (r / 4) + 4 hi + r % 4.
                const uint32_t other = (uint32_t)__shfl_xor((int)seen, 32), s0 = hi ? other : seen, s1 = hi ? seen : other;
                uint32_t sees[2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    sees[t] = ((s0 >> (16 * t)) & 255u) | (((s1 >> (16 * t)) & 255u) << 8) | (((s0 >> (16 * t + 8)) & 255u) << 16) | (((s1 >> (16 * t + 8)) & 255u) << 24);
                const uint32_t map = opaque_vgpr(lds_addr(nan_map[buf][4 * hi]));
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint2_t m2 = *(const lds_uint2 *)lds_ptr(map + (32 * i + 8 * (e >> 2) + (e & 3)) * 8);
                        acc[i][e] = (m2[0] & sees[0]) | (m2[1] & sees[1]) ? NAN : acc[i][e];
                    }
            }
        }
        if (ci + 1 < c1) put(buf ^ 1, ci + 1);           // every wave is past the barrier, and done with that buffer
    }
    if (!rows_here || R.r0 + 32 * wave + col >= R.rows) return;
    l += kvp_other(l);
    const int64_t o = (int64_t)(R.first_token + tok) * c.H * a.G + head;
    const float vs = vref > 0 ? __uint_as_float((uint32_t)vref << 23) : 0.f;      // what the accumulators are relative to
    if (parts > 1) {
        const int64_t at = (((int64_t)tile * c.H + h) * p.splits + split) * KVP_ROWS + 32 * wave + col;   // of records
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (32 * i + 8 * e < D)
                    *(float4_t *)(p.acc + at * D + 32 * i + 8 * e + 4 * hi) =
                        float4_t{acc[i][4 * e] * vs, acc[i][4 * e + 1] * vs, acc[i][4 * e + 2] * vs, acc[i][4 * e + 3] * vs};
        if (hi == 0) *(float2_t *)(p.ml + at * 2) = float2_t{m, l};
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint16_t *out = (uint16_t *)a.out + o * D + 4 * hi;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (32 * i + 8 * e < D) {
                typedef typename mx_type<QT>::T T;
                T v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = (T)(acc[i][4 * e + k] * vs * inv);
                *(uint2_t *)(out + 32 * i + 8 * e) = bitcast<uint2_t>(v);
            }
    if (a.lse && hi == 0) a.lse[o] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * (1.0f / LOG2E);
}

template <int QT, int NT>
static hipError_t launch_kv8_prefill_t(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    constexpr int lds = 2 * kvp_buffer(NT);
    static_assert(lds <= 160 * 1024 - 64, "LDS budget");
    static std::atomic<uint64_t> done{0};
    if (lds > 64 * 1024)
        if (hipError_t e = mx_allow_lds((const void *)kv8_prefill_kernel<QT, NT>, lds, done)) return e;
    hipLaunchKernelGGL((kv8_prefill_kernel<QT, NT>), dim3((unsigned)p.tiles * (unsigned)a.cache.H, (unsigned)p.splits), dim3(64 * KVP_WAVES), lds, s, a, p);
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
