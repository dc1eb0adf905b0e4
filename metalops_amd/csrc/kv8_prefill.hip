// Attention over the 8-bit cache, many rows: tiles of 256 (D > 128: 128) query rows of a key/value
// head (a row is a new token and one of the head's G queries, G neighbouring rows to a token).
//
// Waves with 32 rows each go through the context 64 tokens at a time.  The workgroup turns a
// piece of K and V into 16 bits once, on its way from memory through registers to LDS (two
// buffers each, the next piece's loads in flight during a piece's products; one barrier a piece).
// Both products are v_mfma_f32_32x32x16 with the cache as the A operand, so a lane's results
// belong to one row (l % 32):
//   S^T = K q^T    two tiles of 32 tokens.  A lane holds rows 8 (r / 4) + 4 (l / 32) + r % 4 of a
//                  tile; K's tokens are dealt to the tile's rows so that registers 8 j .. 8 j + 7
//                  are tokens 16 j + 8 (l / 32) .. + 7, and P needs no move between lanes in
//   O^T += V^T P^T whose operand from LDS is 8 such tokens of a channel.
// K lies in LDS token by token, V channel by channel, in rows of an odd number of 16 bytes, so
// that 16 lanes reading 16 rows meet 16 banks.
//
// The exponentials of a piece (VALU) run between the products of the next piece's S (matrix
// cores), for which K is a piece ahead of V in LDS.
//
// Scales, rounding and what is masked are as in kv8_attend.hip: K's scale multiplies the scores
// in fp32; V's is applied by the conversion, relative to the largest one met so far; P is fp16.
// The running maximum follows a row's scores once they exceed it by 2^8 (P stays far below
// fp16's 65504), so that most pieces leave the accumulators alone.
#include <algorithm>
#include <atomic>

#include "kv8_attend.h"

namespace mcq4 {

constexpr int KVP_V_PITCH = KVD_STEP * 2 + 16;
constexpr int kvp_waves(int NT) { return NT <= 4 ? 8 : 4; }
constexpr int kvp_channels(int NT) { return NT <= 4 ? 128 : NT <= 6 ? 192 : 256; }     // in LDS: every thread's part
constexpr int kvp_k_pitch(int NT) { return 2 * kvp_channels(NT) + 16; }
constexpr int kvp_k_bytes(int NT) { return KVD_STEP * kvp_k_pitch(NT); }
constexpr int kvp_v_bytes(int NT) { return kvp_channels(NT) * KVP_V_PITCH; }

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
__global__ void __launch_bounds__(64 * kvp_waves(NT), NT <= 4 ? 2 : 1)
kv8_prefill_kernel(Kv8Attend a, Kv8Plan p) {
    constexpr int WAVES = kvp_waves(NT), ROWS = 32 * WAVES, CH = kvp_channels(NT);
    constexpr int KL = WAVES, NC = CH / (16 * KL);       // threads of a K token; 16-byte pieces of K, and of V, of a thread
    constexpr int K_PITCH = kvp_k_pitch(NT), K_BYTES = kvp_k_bytes(NT), V_BYTES = kvp_v_bytes(NT);
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ int nan_flag[2];
    __shared__ __attribute__((aligned(8))) uint16_t nan_map[2][CH][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hi = lane >> 5;
    // Neighbouring workgroups take neighbouring heads: with 8 of them an XCD's L2 serves one.
    const int h = (int)(blockIdx.x % (uint32_t)a.cache.H), tile = (int)(blockIdx.x / (uint32_t)a.cache.H);
    Kv8Rows R;
    if (!kv8_longest_first(a, tile, ROWS, R)) return;
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
    const int tile_lo = a.window ? R.pos0 + (min(R.r0 + ROWS, R.rows) - 1) / a.G - a.window + 1 : 0;
    auto seen_by_wave = [&](int ci) { return rows_here && ci < c1 && ci * KVD_STEP < any_hi && (ci + 1) * KVD_STEP > any_lo; };

    // A negative scale goes into q's sign: the scores' factor is positive, and a maximum stays one.
    const uint16_t *q = (const uint16_t *)a.q + (int64_t)(R.first_token + tok) * a.q_token + (int64_t)head * a.q_head;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    uint4_t qv[2 * NT];
#pragma unroll
    for (int k = 0; k < 2 * NT; ++k) {
        qv[k] = 16 * k < D ? *(const uint4_t *)(q + 16 * k + 8 * hi) : uint4_t{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) qv[k][e] ^= flip;
    }

    float16_t acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float qk = fabsf(a.scale) * LOG2E;

    // The thread's part of a piece: K token tid / KL (a wave's lie in one page), 16-byte pieces
    // tid % KL + KL i; V channels tid / 4 + 16 WAVES i, tokens 16 (tid % 4) ..  Channels past D
    // repeat the last ones: q is 0 there, and those of V are not stored.  Scale bytes are those
    // of tokens 16 (tid % 4) ..: kb with bit 8 set, vb 0 for a page that is not there.
    // (Made of the thread's number where they are used: registers are short.)
    struct Place { int part, line, k_part, k_line; };
    auto place = [&]() -> Place {
        const int t = (int)opaque_vgpr((uint32_t)tid);
        return {t & 3, t >> 2, t % KL, t / KL};
    };
    uint4_t kr[NC], vr[NC];
    // Table entries: ek, es of the next K to be fetched (its codes, its scales), ev of the next V.
    int ek, es, ev;
    uint32_t kb_next = 0, kb_now = 0, vb_next = 0;
    bool k_there = false, v_there = false;
    int vref = 0, vref_next = 0;
    auto entries = [&](int ci) {
        const Place w = place();
        ev = es;
        ek = kv8_entry(a.batch, page_log, R.b, ci * KVD_STEP + w.k_line);
        es = kv8_entry(a.batch, page_log, R.b, ci * KVD_STEP + 16 * w.part);
    };
    auto fetch_k = [&](int ci) {
        const Place w = place();
        const int t0 = ci * KVD_STEP, idk = kv8_checked(ek, c.P, t0 + (w.k_line & ~15), R.ctx), ids = kv8_checked(es, c.P, t0 + 16 * w.part, R.ctx);
        kb_next = c.ks[(int64_t)max(ids, 0) * c.H + h];
        k_there = ids >= 0;
        const uint8_t *kp = c.k + (((int64_t)max(idk, 0) * c.H + h) * page + ((t0 + w.k_line) & (page - 1))) * D;
#pragma unroll
        for (int i = 0; i < NC; ++i) kr[i] = *(const uint4_t *)(kp + min(16 * (w.k_part + KL * i), D - 16));
    };
    auto fetch_v = [&](int ci) {
        const Place w = place();
        const int t0 = ci * KVD_STEP, id = kv8_checked(ev, c.P, t0 + 16 * w.part, R.ctx);
        const int64_t b = (int64_t)max(id, 0) * c.H + h;
        vb_next = c.vs[b];
        v_there = id >= 0;
        const uint8_t *vp = c.v + b * page * D + ((t0 + 16 * w.part) & (page - 1));
#pragma unroll
        for (int i = 0; i < NC; ++i) vr[i] = *(const uint4_t *)(vp + min(w.line + 16 * WAVES * i, D - 1) * page);
    };
    auto put_k = [&](int buf) {
        const Place w = place();
        uint8_t *kd = smem + buf * K_BYTES + w.k_line * K_PITCH + 32 * w.k_part;
#pragma unroll
        for (int i = 0; i < NC; ++i) kvp_put<QT>(kd + 32 * KL * i, kr[i], 1.0f);
    };
    auto put_v = [&](int buf, int piece) {
        const Place pl = place();
        uint8_t *vd = smem + 2 * K_BYTES + buf * V_BYTES + pl.line * KVP_V_PITCH + 32 * pl.part;
        const int mine = v_there ? (int)vb_next : 0;
        int top = max(mine, __builtin_amdgcn_update_dpp(0, mine, 0xB1, 0xF, 0xF, true));     // lanes 1 0 3 2
        top = max(top, __builtin_amdgcn_update_dpp(0, top, 0x4E, 0xF, 0xF, true));           // lanes 2 3 0 1
        vref_next = max(vref_next, __builtin_amdgcn_readfirstlane(top));
        const int rel = mine - vref_next;
        const float vs = rel < -100 ? 0x1p-100f : __uint_as_float((uint32_t)(rel + 127) << 23);
        if (!__all(v_there)) {                               // what page 0 holds there is not seen
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (!v_there) vr[i] = uint4_t{0, 0, 0, 0};
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
                nan_map[buf][pl.line + 16 * WAVES * i][pl.part] = (uint16_t)map;
                if (map) nan_flag[buf] = piece + 1;
            }
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) kvp_put<DT_F16>(vd + 16 * WAVES * i * KVP_V_PITCH, vr[i], vs);
    };

    // K row of S-tile row l % 32: rows 16 j + 8 e + 4 h + i are tokens 16 j + 8 h + 4 e + i.
    const int k_row = (col & 16) | ((col & 4) << 1) | ((col & 8) >> 1) | (col & 3);
    const uint32_t lds0 = lds_addr(smem);
    const uint32_t k_off = lds0 + k_row * K_PITCH + 16 * hi, v_off = lds0 + 2 * K_BYTES + col * KVP_V_PITCH + 16 * hi;
    auto read_k = [&](int buf, int i) { return mx_lds16(k_off + buf * K_BYTES + 32 * (i & 1) * K_PITCH + 32 * (i >> 1)); };       // i = 2 k + t
    auto read_v = [&](int buf, int i) { return mx_lds16(v_off + buf * V_BYTES + 32 * (i % NT) * KVP_V_PITCH + 32 * (i / NT)); };  // i = NT (2 t + j) + channel tile

    // A piece's raw scores; by 16 tokens the factor that makes them logarithms to base 2 (never
    // 0: masked ones are -inf); which of them the row sees (bit 16 t + e: s[t][e]); their maximum.
    float16_t s[2], sn[2], zero;
#pragma unroll
    for (int e = 0; e < 16; ++e) zero[e] = 0.f;
    float ks[4] = {0.f, 0.f, 0.f, 0.f}, mx = -INFINITY;
    uint32_t seen = ~0u;
    auto finish = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        uint32_t kb[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            kb[g] = (uint32_t)__builtin_amdgcn_readlane((int)kb_now, g);
            ks[g] = fmaxf(qk * __uint_as_float((kb[g] & 255u) << 23), 0x1p-126f);
        }
        seen = ~0u;
        if (t0 < all_lo || t0 + KVD_STEP > all_hi || ((kb[0] | kb[1] | kb[2] | kb[3]) & 256u)) {
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
        mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float x = s[g >> 1][8 * (g & 1)];
#pragma unroll
            for (int e = 1; e < 8; ++e) x = fmaxf(x, s[g >> 1][8 * (g & 1) + e]);
            mx = fmaxf(mx, x * ks[g]);
        }
        mx = fmaxf(mx, kvp_other(mx));
    };

    if (tid < 2) nan_flag[tid] = 0;                      // piece + 1 where a buffer's V has a NaN
    if (c0 < c1) {
        es = 0;
        entries(c0);
        fetch_k(c0);
        entries(c0 + 1);
        put_k(0);
        kb_now = k_there ? kb_next : 256u;
        fetch_k(c0 + 1);
        fetch_v(c0);
        entries(c0 + 2);
        __syncthreads();
        if (seen_by_wave(c0)) {
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) s[i & 1] = kvp_mfma<QT>(read_k(0, i), qv[i >> 1], i < 2 ? zero : s[i & 1]);
            finish(c0);
        }
        put_k(1);
        put_v(0, c0);
        kb_now = k_there ? kb_next : 256u;
    }
    wait_vmcnt<0>();                                     // q too: nothing in the loop waits for it again
    for (int ci = c0; ci < c1; ++ci) {
        const int buf = (ci - c0) & 1, top = vref_next;
        if (ci + 1 < c1) {
            fetch_k(ci + 2);
            fetch_v(ci + 1);
            entries(ci + 3);
        }
        lds_barrier();                                   // V of the piece and K of the next are there, the other buffers have been read
        const bool has_nan = nan_flag[buf] == ci + 1;
        if (seen_by_wave(ci)) {
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
            // 4 NT products of the next S, and 16 pairs of weights between them; operands are read AHEAD products early.
            constexpr int AHEAD = 2, N1 = 4 * NT;
            uint4_t pr[4], op[AHEAD];
            float add[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) op[i] = read_k(buf ^ 1, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < N1; ++i) {
                sn[i & 1] = kvp_mfma<QT>(op[i % AHEAD], qv[i >> 1], i < 2 ? zero : sn[i & 1]);
                if (i + AHEAD < N1) op[i % AHEAD] = read_k(buf ^ 1, i + AHEAD);
#pragma unroll
                for (int w = 0; w < 16; ++w)
                    if (w * N1 / 16 == i) {
                        const int g = w >> 2, t = g >> 1, e = 8 * (g & 1) + 2 * (w & 3);
                        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], ks[g], -m_use));
                        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e + 1], ks[g], -m_use));
                        add[w & 1] += x + y;
                        pr[g][w & 3] = bitcast<uint32_t>(half2_t{(_Float16)x, (_Float16)y});
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
            l += add[0] + add[1];
            uint4_t ov[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) ov[i] = read_v(buf, i);
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) {
                acc[i % NT] = kvp_mfma<DT_F16>(ov[i % AHEAD], pr[i / NT], acc[i % NT]);
                if (i + AHEAD < 4 * NT) ov[i % AHEAD] = read_v(buf, i + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
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
        } else if (seen_by_wave(ci + 1)) {
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) sn[i & 1] = kvp_mfma<QT>(read_k(buf ^ 1, i), qv[i >> 1], i < 2 ? zero : sn[i & 1]);
        }
        if (ci + 1 < c1) {
            // Every wave is past the barrier, and done with these buffers.
            put_k(buf);
            put_v(buf ^ 1, ci + 1);
            s[0] = sn[0];
            s[1] = sn[1];
            if (seen_by_wave(ci + 1)) finish(ci + 1);
            kb_now = k_there ? kb_next : 256u;
        }
    }
    if (!rows_here || R.r0 + 32 * wave + col >= R.rows) return;
    l += kvp_other(l);
    const int64_t o = (int64_t)(R.first_token + tok) * c.H * a.G + head;
    const float vs = vref > 0 ? __uint_as_float((uint32_t)vref << 23) : 0.f;      // what the accumulators are relative to
    if (parts > 1) {
        const int64_t at = (((int64_t)tile * c.H + h) * p.splits + split) * ROWS + 32 * wave + col;   // of records
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
    constexpr int lds = 2 * (kvp_k_bytes(NT) + kvp_v_bytes(NT));
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
