// Attention over the 8-bit cache, few rows: softmax(scale q k^T) v for the 16 (or fewer) query
// rows that share a key/value head, a row being a new token and one of the head's G queries.
//
// A wave takes 64 tokens at a time, K and V from memory to registers in 16-byte loads, and
// keeps the running maximum and sum of its rows.  Both products are v_mfma_f32_16x16x32 with
// the cache as the A operand, so a lane's results belong to one row (column l % 16):
//   S^T = K q^T    four tiles of 16 tokens.  Row r of tile a is token 16 (r / 4) + 4 a + r % 4,
//                  so lane group g = l / 16 ends up with tokens 16 g .. 16 g + 15, which lie in
//                  one page: one scale for the lane, and
//   O^T += V^T P^T takes P as it lies in registers: a lane of V^T holds 16 consecutive tokens
//                  16 g .. of one channel, one 16-byte load.
// e4m3 becomes 16 bits exactly (v_cvt_scalef32_pk_*_fp8).  K's scale multiplies the scores in
// fp32, V's goes into P (kv8_attend.h): relative to the largest scale that the wave meets instead,
// in the conversion of V, a page that a row does not see, or that has no weight in it, would take
// the row's others out of fp16's range.  P is rounded to fp16; its largest stands at 2^15, so that
// weights down to 2^-29 of it have 11 bits (relative to 1 those below 2^-25 would be 0, and a row
// whose first token takes the weight would lose its others).
//
// A masked score is -inf whatever K holds there, but 0 times a NaN of V would be NaN: tiles with
// a masked token look for NaN codes, zero them, and set the rows that do attend to one to NaN.
//
// Contexts differ in length, so a workgroup does not get a sequence or a fixed part of one: the
// pieces of 64 tokens of all tiles of all heads stand in one row, and each workgroup takes an
// equal stretch of it (kv8_share), in it one tile after another, four waves with every fourth
// piece.  As many workgroups as the CUs hold at once then end together: 32 sequences of 1 to
// 8192 tokens took 105 us in parts of 16 pieces and 89 in parts of 64.  A tile that lies
// in one stretch is finished there; of others each stretch leaves a record, at most two a
// workgroup, draws a ticket of the workgroup in which the tile begins, and the last of them adds
// the records up in their order.
//
// Bound by memory where contexts are long: 32 sequences of 1 to 8192 tokens (8 heads of keys,
// D = 128, 252 MB) take 62 us, 4.1 TB/s against 4.9 of a large copy.  One token behind 32768
// (67 MB) takes 23: a workgroup has two pieces a wave, so the chain from the contexts' sums over the
// table to the first pieces, and the join, are half of it (a join kernel of its own made it 25).
#include <algorithm>
#include <atomic>
#include <stdlib.h>

#include "kv8_attend.h"

namespace mcq4 {

constexpr int KVD_WAVES = 4;
// P's largest, 2^15, stays below fp16's 65504.
constexpr int KVD_P_LOG = 15;

// Pieces of a tile; a tile without any counts as one, so that its rows are written.  All pieces of
// all heads fit 31 bits (kv8_plan), if no token is two sequences'.
__device__ __forceinline__ int kv8_pieces(const Kv8Rows &R) { return max(1, R.hi - R.lo); }
__device__ __forceinline__ int kv8_seq_pieces(const Kv8Attend &a, int b) {
    int n = 0;
    Kv8Rows R;
    for (int i = 0; kv8_tile(a, b, i, KVD_ROWS, R); ++i) n += kv8_pieces(R);
    return n;
}
// A workgroup's stretch: pieces [start, end) of all heads', the first of them in sequence b of head
// h, which begins at `at`.  Every lane of the wave takes part.
struct Kv8Share { int start, end, chunk, h, b, at; };
__device__ __forceinline__ Kv8Share kv8_share(const Kv8Attend &a, const Kv8Plan &p) {
    const int lane = threadIdx.x & 63, B = a.batch.B;
    auto add = [](uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); };
    auto scan = [&](uint32_t v) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d);
            if (lane >= d) v = add(v, up);
        }
        return v;
    };
    int own = lane < B ? kv8_seq_pieces(a, lane) : 0, sum = (int)scan(own);
    uint32_t total = __shfl(sum, 63);
    for (int b0 = 64; b0 < B; b0 += 64) total = add(total, __shfl(scan(b0 + lane < B ? kv8_seq_pieces(a, b0 + lane) : 0), 63));
    Kv8Share o = {};
    // Offsets that fall and rise again can give a token to many sequences, and more pieces than 31 bits count: none is taken.
    if (total == 0 || (uint64_t)total * (uint32_t)a.cache.H > 0x7FFFFFFFu) return o;
    const int per_head = (int)total, all = per_head * a.cache.H;
    // At least a piece for each wave, unless that would string short contexts together.
    const int least = p.chunk ? p.chunk : min(KVD_WAVES, (per_head + B - 1) / B);
    o.chunk = max((int)(((uint32_t)all + p.wgs - 1) / p.wgs), least);
    const int64_t start = (int64_t)blockIdx.x * o.chunk;
    if (start >= all) return o;
    o.start = (int)start;
    o.end = (int)min(start + o.chunk, (int64_t)all);
    o.h = o.start / per_head;
    const int in_head = o.start - o.h * per_head;
    int before = 0;
    for (int b0 = 0;;) {
        const uint64_t past = __ballot(before + sum > in_head);
        if (past) {
            const int l = __builtin_ctzll(past);
            o.b = b0 + l;
            o.at = o.h * per_head + before + __shfl(sum, l) - __shfl(own, l);
            return o;
        }
        before += __shfl(sum, 63);
        b0 += 64;
        if (b0 >= B) return Kv8Share{};             // not reached
        own = b0 + lane < B ? kv8_seq_pieces(a, b0 + lane) : 0;
        sum = (int)scan(own);
    }
}

// The records: accumulators [records][rows][D], then maxima and sums.  They are written and read at agent scope, past
// the XCDs' L2s, which are not coherent.
constexpr int KVD_AGENT = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv8_records(const Kv8Plan &p, int D) {
    return mx_rsrc(p.acc, (int64_t)p.records * KVD_ROWS * (D + 2) * 4);
}

// The prefix's part in four channels of row o of q: its records in order, then the row's own sums.
__device__ __forceinline__ void kv8_with_prefix(const Kv8Attend &a, int64_t o, int d, float4_t &v, float &top, float &l) {
    constexpr int BATCH = 8;
    const Kv8Prefix &x = a.pre;
    const int2 at = x.at[o];
    const int D = a.cache.D;
    int parts = max(at.y, 0);
    if (at.x < 0 || at.x + (int64_t)(parts - 1) * x.rows >= x.records * x.rows) parts = 0;      // groups that fall: no records of this row
    float m = -INFINITY, sum = 0.f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += BATCH) {
        float2_t ml[BATCH];
        float4_t part[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t row = at.x + (int64_t)min(s0 + i, parts - 1) * x.rows;
            ml[i] = *(const float2_t *)(x.ml + row * 2);
            part[i] = *(const float4_t *)(x.acc + row * D + d);
        }
        float most = m;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) most = fmaxf(most, ml[i][0]);
        const float use = most == -INFINITY ? 0.f : most, shrink = __builtin_amdgcn_exp2f(m - use);
        m = most;
        sum *= shrink;
        acc *= shrink;
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (s0 + i < parts) {
                const float w = __builtin_amdgcn_exp2f(ml[i][0] - use);
                sum += ml[i][1] * w;
                acc += part[i] * w;
            }
    }
    const float most = fmaxf(m, top), use = most == -INFINITY ? 0.f : most;
    const float w0 = __builtin_amdgcn_exp2f(m - use), w1 = __builtin_amdgcn_exp2f(top - use);
    v = acc * w0 + v * w1;
    l = sum * w0 + l * w1;
    top = most;
}

// Four channels of row rr of a tile, from their sum with its maximum and sum of weights.
template <int QT>
__device__ __forceinline__ void kv8_write(const Kv8Attend &a, const Kv8Rows &R, int h, int rr, int d, float4_t v, float top, float l) {
    const int rt = (R.r0 + rr) / a.G, rh = h * a.G + (R.r0 + rr) % a.G;
    const int64_t o = (int64_t)(R.first_token + rt) * a.cache.H * a.G + rh;
    const float inv = l == 0.f ? 0.f : 1.0f / l;            // a row that sees nothing is 0
#pragma unroll
    for (int e = 0; e < 4; ++e) mx_store<QT>(a.out, o * a.cache.D + d + e, v[e] * inv);
    if (a.lse && d == 0) a.lse[o] = l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * (1.0f / LOG2E);
}

template <int QT, int NH>
__device__ __forceinline__ void kv8_attend_tile(const Kv8Attend &a, const Kv8Plan &p, const Kv8Rows &R, int h, int c0, int c1, int record,
                                                uint8_t *smem) {
    constexpr int ND = 4 * NH;                      // channel tiles of 16
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const Kv8Cache &c = a.cache;
    const int D = c.D, page_log = c.page_log, page = 1 << page_log;
    // This lane's row.
    const int r = min(R.r0 + col, R.rows - 1);
    const int tok = r / a.G, head = h * a.G + r % a.G;
    const int pos = R.pos0 + tok;
    const int see_hi = a.causal ? min(pos + 1, R.ctx) : R.ctx;
    const int see_lo = a.window ? max(pos - a.window + 1, 0) : 0;
    // Tokens that every row of the tile sees.
    const int tok_a = R.r0 / a.G, tok_z = (min(R.r0 + KVD_ROWS, R.rows) - 1) / a.G;
    const int all_hi = a.causal ? R.pos0 + tok_a + 1 : R.ctx, all_lo = a.window ? R.pos0 + tok_z - a.window + 1 : 0;

    const uint16_t *q = (const uint16_t *)a.q + (int64_t)(R.first_token + tok) * a.q_token + (int64_t)head * a.q_head;
    uint4_t qv[NH][2];
#pragma unroll
    for (int i = 0; i < NH; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int d = 64 * i + 16 * g + 8 * u;
            qv[i][u] = d < D ? *(const uint4_t *)(q + d) : uint4_t{0, 0, 0, 0};
        }

    float4_t acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    float part = -INFINITY, k = KV8_NO_K;           // the largest s - m + v, and k
    const float qk = a.scale * LOG2E;

    const int k_sub = 16 * (col >> 2) + (col & 3);  // K row of tile a: token k_sub + 4 a
    uint4_t kr[4][NH], vr[ND];
    // A piece's K and V go out as soon as the registers of the one before are free, its page
    // numbers an iteration earlier.  Groups without tokens read page 0, whose bytes are not used.
    int ek = 0, ev = 0, pv = -1;
    auto pages = [&](int ci) {
        const int tk = ci * KVD_STEP + 16 * (col >> 2), tv = ci * KVD_STEP + 16 * g;
        ek = kv8_entry(a.batch, page_log, R.b, tk);
        ev = kv8_entry(a.batch, page_log, R.b, tv);
    };
    uint32_t kb = 0, vb = 0;
    auto fetch_k = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        const int pk = kv8_checked(ek, c.P, t0 + 16 * (col >> 2), R.ctx);
        pv = kv8_checked(ev, c.P, t0 + 16 * g, R.ctx);
        const int64_t bk = (int64_t)max(pk, 0) * c.H + h, bv = (int64_t)max(pv, 0) * c.H + h;
        kb = c.ks[bv];
        vb = c.vs[bv];
        const uint8_t *kp = c.k + bk * page * D + (int64_t)((t0 + k_sub) & (page - 1)) * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < NH; ++i)
                kr[t][i] = *(const uint4_t *)(kp + 4 * t * D + min(64 * i + 16 * g, D - 16));      // past D: q is 0
    };
    auto fetch_v = [&](int ci) {
        const int64_t bv = (int64_t)max(pv, 0) * c.H + h;
        const uint8_t *vp = c.v + bv * page * D + (int64_t)col * page + ((ci * KVD_STEP + 16 * g) & (page - 1));
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D) vr[i] = *(const uint4_t *)(vp + (int64_t)16 * i * page);
    };

    if (c0 + wave < c1) {
        pages(c0 + wave);
        fetch_k(c0 + wave);
        fetch_v(c0 + wave);
        pages(c0 + wave + KVD_WAVES);
    }
    for (int ci = c0 + wave; ci < c1; ci += KVD_WAVES) {
        const bool more = ci + KVD_WAVES < c1;
        // A page that is not there: nothing of it is seen.
        const bool here = pv >= 0;
        const float kscale = here && kb < 255 ? qk * __uint_as_float(kb << 23) : NAN;
        const bool v_nan = here && vb == 255;
        const float vbyte = here ? (float)vb : 0.f;
        const int t0 = ci * KVD_STEP, t_own = t0 + 16 * g;
        float4_t s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NH; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    s[t] = mx_mfma16<QT>(kv8_eight<QT>(kr[t][i][2 * u], kr[t][i][2 * u + 1], 1.0f), qv[i][u], s[t]);
        }
        if (more) fetch_k(ci + KVD_WAVES);
        const bool full = t0 >= all_lo && t0 + KVD_STEP <= all_hi && __all(here);
        float mx = -INFINITY;
        uint32_t seen = 0xFFFFu;                    // bit 4 t + i: the row sees token t_own + 4 t + i
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = s[t][i] * kscale;
                if (!full) {
                    const int at = t_own + 4 * t + i;
                    const bool sees = here && at < see_hi && at >= see_lo;
                    v = sees ? v : -INFINITY;
                    if (!sees) seen &= ~(1u << (4 * t + i));
                }
                s[t][i] = v;
                mx = fmaxf(mx, v);
            }
        const float m_new = fmaxf(m, kv8_group_max(mx)), m_use = m_new == -INFINITY ? 0.f : m_new, drop = m - m_use;
        part = fmaxf(part + drop, kv8_group_max(mx - m_use + vbyte));
        const float k_new = ceilf(kv8_k(part)), shrink = __builtin_amdgcn_exp2f(drop + (k - k_new));
        const float log = fmaxf(vbyte - k_new + KVD_P_LOG, KV8_LEAST);
        float base = m_use - log;
        if (__any(fabsf(m_use) >= KV8_HUGE)) {
#pragma unroll
            for (int t = 0; t < 4; ++t) s[t] -= m_use;
            base = -log;
        }
        m = m_new;
        k = k_new;
        float add = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - base);
                add += s[t][i];
            }
        l = l * __builtin_amdgcn_exp2f(drop) + __builtin_ldexpf(add, -(int)log);
        uint4_t pr[2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            pr[t >> 1][2 * (t & 1)] = bitcast<uint32_t>(half2_t{(_Float16)s[t][0], (_Float16)s[t][1]});
            pr[t >> 1][2 * (t & 1) + 1] = bitcast<uint32_t>(half2_t{(_Float16)s[t][2], (_Float16)s[t][3]});
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] *= shrink;
        if (__any(v_nan)) {                         // byte 255: every value of the page
#pragma unroll
            for (int i = 0; i < ND; ++i)
                if (v_nan) vr[i] = uint4_t{0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu};
        }
        uint32_t bad = 0;
        if (!full) {
#pragma unroll
            for (int i = 0; i < ND; ++i)
                if (16 * i < D)
#pragma unroll
                    for (int w = 0; w < 4; ++w) bad |= kv8_nan_bytes(vr[i][w]);
        }
        if (__any(bad != 0)) {
            // NaN of V: counted per row and channel by a product of ones, and taken out.
            uint4_t pn[2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    pn[t >> 1][2 * (t & 1) + i] = ((seen >> (4 * t + 2 * i)) & 1 ? 0x3C00u : 0u) | ((seen >> (4 * t + 2 * i + 1)) & 1 ? 0x3C000000u : 0u);
#pragma unroll
            for (int i = 0; i < ND; ++i)
                if (16 * i < D) {
                    uint4_t n;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t f = here ? kv8_nan_bytes(vr[i][w]) : 0u;
                        n[w] = f & 0x38383838u;                       // e4m3's 1.0
                        vr[i][w] &= here ? ~f : 0u;
                    }
                    float4_t count = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < 2; ++u) count = mx_mfma16<DT_F16>(kv8_eight<DT_F16>(n[2 * u], n[2 * u + 1], 1.0f), pn[u], count);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (count[e] > 0.f) acc[i][e] = NAN;
                }
        }
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    acc[i] = mx_mfma16<DT_F16>(kv8_eight<DT_F16>(vr[i][2 * u], vr[i][2 * u + 1], 1.0f), pr[u], acc[i]);
        if (more) {
            fetch_v(ci + KVD_WAVES);
            pages(ci + 2 * KVD_WAVES);
        }
    }
    l = kv8_group_sum(l);

    // The waves' parts: maxima, sums and scaled accumulators, [wave][row], in LDS.
    const int pitch = D + 4;
    float *wm = (float *)smem, *wl = wm + KVD_WAVES * 16, *wacc = wl + KVD_WAVES * 16;      // [wave][16][pitch]
    if (g == 0) { wm[wave * 16 + col] = m; wl[wave * 16 + col] = l; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < KVD_WAVES; ++w) top = fmaxf(top, wm[w * 16 + col]);
    const float t_use = top == -INFINITY ? 0.f : top;
    const Kv8Power unit(fmaxf(m - t_use + k - (KVD_P_LOG + 127), -2000.f));
    float *mine = wacc + (wave * 16 + col) * pitch + 4 * g;
#pragma unroll
    for (int i = 0; i < ND; ++i)
        if (16 * i < D) *(float4_t *)(mine + 16 * i) = unit * acc[i];
    __syncthreads();
    const int rows = min(KVD_ROWS, R.rows - R.r0), D4 = D >> 2;
    for (int i = threadIdx.x; i < rows * D4; i += 64 * KVD_WAVES) {
        const int rr = i / D4, d = 4 * (i % D4);
        float tm = -INFINITY, tl = 0.f;
#pragma unroll
        for (int w = 0; w < KVD_WAVES; ++w) tm = fmaxf(tm, wm[w * 16 + rr]);
        const float tu = tm == -INFINITY ? 0.f : tm;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KVD_WAVES; ++w) {
            tl += wl[w * 16 + rr] * __builtin_amdgcn_exp2f(wm[w * 16 + rr] - tu);
            v += *(const float4_t *)(wacc + (w * 16 + rr) * pitch + d);
        }
        if (record >= 0) {
            const int at = record * KVD_ROWS + rr;
            __builtin_amdgcn_raw_buffer_store_b128(bitcast<uint4_t>(v), kv8_records(p, D), (at * D + d) * 4, 0, KVD_AGENT);
            if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(bitcast<uint2_t>(float2_t{tm, tl}), kv8_records(p, D), (p.records * KVD_ROWS * D + 2 * at) * 4, 0, KVD_AGENT);
        } else {
            kv8_write<QT>(a, R, h, rr, d, v, tm, tl);
        }
    }
}

// The records of a tile of `parts` stretches, the first of them that of workgroup `begun`, added up in order by the
// last workgroup that wrote one.  A thread takes four channels of a row and, where that leaves threads over, every
// groups-th part; their sums are added in the end.
constexpr int KVJ_LOADS = 16;
template <int QT>
__device__ __forceinline__ void kv8_join_tile(const Kv8Attend &a, const Kv8Plan &p, const Kv8Rows &R, int h, int begun, int slot, int parts, uint8_t *smem) {
    constexpr int THREADS = 64 * KVD_WAVES;
    float4_t *gacc = (float4_t *)smem;              // [THREADS]
    float2_t *gml = (float2_t *)(gacc + THREADS);
    const int tid = threadIdx.x, D = a.cache.D, D4 = D >> 2, rows = min(KVD_ROWS, R.rows - R.r0), units = rows * D4;
    const int groups = max(1, min(parts, THREADS / units));
    const __amdgpu_buffer_rsrc_t rs = kv8_records(p, D);
    for (int u0 = 0; u0 < units; u0 += THREADS) {
        const int gr = groups == 1 ? 0 : tid / units, u = u0 + (groups == 1 ? tid : tid % units);
        const bool on = u < units && gr < groups;
        const int rr = on ? u / D4 : 0, d = on ? 4 * (u % D4) : 0;
        float top = -INFINITY, l = 0.f;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = min(gr, groups - 1); s0 < parts; s0 += groups * KVJ_LOADS) {
            uint4_t x[KVJ_LOADS];
            uint2_t ml[KVJ_LOADS];
#pragma unroll
            for (int i = 0; i < KVJ_LOADS; ++i) {
                const int s = min(s0 + i * groups, parts - 1), at = (s ? 2 * (begun + s) : 2 * begun + slot) * KVD_ROWS + rr;
                ml[i] = __builtin_amdgcn_raw_buffer_load_b64(rs, (p.records * KVD_ROWS * D + 2 * at) * 4, 0, KVD_AGENT);
                x[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (at * D + d) * 4, 0, KVD_AGENT);
            }
            float most = top;
#pragma unroll
            for (int i = 0; i < KVJ_LOADS; ++i) most = fmaxf(most, __uint_as_float(ml[i][0]));       // the last part's again, if fewer
            const float use = most == -INFINITY ? 0.f : most, shrink = __builtin_amdgcn_exp2f(top - use);
            top = most;
            l *= shrink;
            v *= shrink;
#pragma unroll
            for (int i = 0; i < KVJ_LOADS; ++i)
                if (s0 + i * groups < parts) {
                    const float w = __builtin_amdgcn_exp2f(__uint_as_float(ml[i][0]) - use);
                    l += __uint_as_float(ml[i][1]) * w;
                    v += bitcast<float4_t>(x[i]) * w;
                }
        }
        if (groups > 1) {
            gacc[tid] = v;
            gml[tid] = float2_t{top, l};
            __syncthreads();
            if (on && gr == 0) {
                for (int i = 1; i < groups; ++i) top = fmaxf(top, gml[tid + i * units][0]);
                const float use = top == -INFINITY ? 0.f : top;
                v *= __builtin_amdgcn_exp2f(gml[tid][0] - use);
                l *= __builtin_amdgcn_exp2f(gml[tid][0] - use);
                for (int i = 1; i < groups; ++i) {
                    const float2_t ml = gml[tid + i * units];
                    const float w = __builtin_amdgcn_exp2f(ml[0] - use);
                    v += gacc[tid + i * units] * w;
                    l += ml[1] * w;
                }
            }
        }
        if (on && gr == 0) kv8_write<QT>(a, R, h, rr, d, v, top, l);
    }
}

template <int QT, int NH>
__global__ void __launch_bounds__(64 * KVD_WAVES, NH <= 2 ? 2 : 1)
kv8_attend_kernel(Kv8Attend a, Kv8Plan p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    kv8_rest(a, blockIdx.x, gridDim.x);
    Kv8Share sh = kv8_share(a, p);
    sh = {kv8_same(sh.start), kv8_same(sh.end), kv8_same(sh.chunk), kv8_same(sh.h), kv8_same(sh.b), kv8_same(sh.at)};
    __shared__ int last;
    int h = sh.h, b = sh.b, i = 0, at = sh.at;      // at: of tile i of sequence b
    while (at < sh.end) {
        Kv8Rows R;
        if (!kv8_tile(a, b, i, KVD_ROWS, R)) {      // the sequence's last tile was the one before
            i = 0;
            if (++b < a.batch.B) continue;
            b = 0;
            if (++h == a.cache.H) break;
            continue;
        }
        kv8_uniform(R);
        const int n = kv8_pieces(R), from = max(sh.start - at, 0), to = min(sh.end - at, n);
        if (from < to) {
            const int slot = at + from > sh.start ? 1 : 0;
            const bool whole = from == 0 && to == n;
            kv8_attend_tile<QT, NH>(a, p, R, h, R.lo + from, min(R.lo + to, R.hi), whole ? -1 : 2 * (int)blockIdx.x + slot, smem);
            if (!whole) __builtin_amdgcn_s_waitcnt(0x0F70);          // vmcnt(0): the record is in memory
            __syncthreads();                        // the waves' parts in LDS have been read
            if (!whole) {
                const int begun = at / sh.chunk, parts = (at + n - 1) / sh.chunk - begun + 1;
                if (threadIdx.x == 0) {
                    last = __hip_atomic_fetch_add(&p.tickets[begun], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1;
                    if (last) __hip_atomic_store(&p.tickets[begun], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (last) kv8_join_tile<QT>(a, p, R, h, begun, at > begun * sh.chunk ? 1 : 0, parts, smem);
                __syncthreads();
            }
        }
        at += n;
        ++i;
    }
}

// Large tiles: the records of 16 rows added up in order.  The workgroup's threads are dealt out over the rows'
// channels, four each, and where that leaves some over, over every groups-th part, whose sums are added in the end.
// PREFIX: with a prefix's records behind them (a kernel of its own: its registers cost the other a quarter).
constexpr int KVJ_THREADS = 256, KVJ_BATCH = 8, KVJ_ROWS = 16;
template <int QT, bool PREFIX>
__global__ void __launch_bounds__(KVJ_THREADS)
kv8_join_kernel(Kv8Attend a, Kv8Plan p) {
    const Kv8Cache &c = a.cache;
    __shared__ __attribute__((aligned(16))) float4_t gacc[KVJ_THREADS];
    __shared__ float gl[KVJ_THREADS];
    extern __shared__ __attribute__((aligned(16))) float2_t mls[];         // [rows][parts]
    const int D4 = c.D >> 2, tid = threadIdx.x, h = blockIdx.y;
    const int tile = blockIdx.x / (p.rows / KVJ_ROWS), rr0 = blockIdx.x % (p.rows / KVJ_ROWS) * KVJ_ROWS;
    Kv8Rows R;
    if (!kv8_longest_first(a, tile, p.rows, R) || R.r0 + rr0 >= R.rows) return;
    const int parts = kv8_parts(R, p);
    if (parts <= 1 && !PREFIX) return;                                     // written by its only part
    const int base = (tile * c.H + h) * p.splits, rows = min(KVJ_ROWS, R.rows - R.r0 - rr0);
    auto record = [&](int s) { return (int64_t)(base + s) * p.rows + rr0; };
    for (int i = tid; i < rows * parts; i += KVJ_THREADS) mls[i % rows * parts + i / rows] = *(const float2_t *)(p.ml + (record(i / rows) + i % rows) * 2);
    __syncthreads();
    const int units = rows * D4;
    const int groups = max(1, min(parts, KVJ_THREADS / units));
    for (int u0 = 0; u0 < units; u0 += KVJ_THREADS) {
        const int gr = groups == 1 ? 0 : tid / units, u = u0 + (groups == 1 ? tid : tid % units);
        const bool on = u < units && gr < groups;
        const int rr = u / D4, d = 4 * (u % D4);
        float top = -INFINITY, l = 0.f;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        if (on) {
            const float2_t *ml = mls + rr * parts;
            for (int s = 0; s < parts; ++s) top = fmaxf(top, ml[s][0]);
            const float use = top == -INFINITY ? 0.f : top;
            for (int s0 = gr; s0 < parts; s0 += groups * KVJ_BATCH) {
                float4_t x[KVJ_BATCH];
#pragma unroll
                for (int i = 0; i < KVJ_BATCH; ++i)
                    x[i] = *(const float4_t *)(p.acc + (record(min(s0 + i * groups, parts - 1)) + rr) * c.D + d);
#pragma unroll
                for (int i = 0; i < KVJ_BATCH; ++i) {
                    const int s = s0 + i * groups;
                    if (s >= parts) break;
                    const float w = __builtin_amdgcn_exp2f(ml[s][0] - use);
                    l += ml[s][1] * w;
                    v += x[i] * w;
                }
            }
        }
        if (groups > 1) {
            gacc[tid] = v;
            gl[tid] = l;
            __syncthreads();
            if (on && gr == 0)
                for (int i = 1; i < groups; ++i) {
                    v += gacc[tid + i * units];
                    l += gl[tid + i * units];
                }
        }
        if (!on || gr) continue;
        if constexpr (PREFIX) {
            const int r = R.r0 + rr0 + rr, tok = r / a.G;
            // A row that stands before its own context sees nothing of the prefix either.
            if (R.pos0 + tok >= 0) kv8_with_prefix(a, ((int64_t)(R.first_token + tok) * c.H + h) * a.G + r % a.G, d, v, top, l);
        }
        kv8_write<QT>(a, R, h, rr0 + rr, d, v, top, l);
    }
}

static Kv8Plan kv8_plan(const Kv8Attend &a) {
    Kv8Plan p;
    const Kv8Batch &b = a.batch;
    const int64_t avg_rows = b.cu ? (int64_t)b.T * a.G / b.B : (int64_t)b.each * a.G;
    int64_t seen = std::min<int64_t>((int64_t)b.W << a.cache.page_log, a.max_context);
    if (a.window && !b.cu) seen = std::min<int64_t>(seen, (int64_t)a.window + b.each + 2 * KVD_STEP);
    const int64_t pieces = std::max<int64_t>(1, (seen + KVD_STEP - 1) / KVD_STEP);
    p.rows = avg_rows > 32 || a.pre.at ? kvp_rows(a.cache.D) : KVD_ROWS;      // a prefix is added where large tiles' parts are
    if (const char *v = opt("MCQ4_KV8_ROWS")) p.rows = atoi(v) > KVD_ROWS || a.pre.at ? kvp_rows(a.cache.D) : KVD_ROWS;
    // The kernel of few rows counts the pieces of all its tiles in 31 bits, whatever the contexts turn out to be.
    const int64_t table_pieces = ((int64_t)b.W << a.cache.page_log) / KVD_STEP + 2, tiles16 = (int64_t)b.T * a.G / KVD_ROWS + b.B;
    if (table_pieces * tiles16 > ((int64_t)1 << 31) / a.cache.H - 1) p.rows = kvp_rows(a.cache.D);
    p.tiles = b.cu ? (int)(((int64_t)b.T * a.G) / p.rows + b.B) : b.B * ((b.each * a.G + p.rows - 1) / p.rows);
    const int64_t wgs = (int64_t)p.tiles * a.cache.H;
    const char *forced = opt("MCQ4_KV8_SPAN");
    p.splits = p.span = p.wgs = p.chunk = p.records = 0;
    if (p.rows == KVD_ROWS) {
        // As many workgroups as the CUs hold at once: two each, or one where D > 128 takes the registers.
        const int64_t most = wgs * pieces;
        p.wgs = (int)std::min<int64_t>(a.cache.D <= 128 ? 512 : 256, most);
        if (forced) {
            p.chunk = std::max(1, atoi(forced));
            p.wgs = (int)std::min<int64_t>((most + p.chunk - 1) / p.chunk, 1024);
        }
        // No tile is divided where there is one stretch, or no context can be longer than a piece (max_context is not
        // relied on for that).
        p.records = p.wgs == 1 || ((int64_t)b.W << a.cache.page_log) <= KVD_STEP ? 0 : 2 * p.wgs;
    } else {
        // A CU holds one workgroup, so parts that make 256 of them, of four pieces at least: 256 tokens of 16384
        // (32 heads, 8 of keys, D = 128) 97 us in parts of 32 pieces, 116 in parts of 16, 151 in parts of 64; 64 of
        // 8192 43 in parts of 4, 47 in parts of 8.  Tiles that are 256 by themselves stay whole (2048 of 2048: 80,
        // in halves 84).
        int64_t span = forced ? std::max(1, atoi(forced)) : wgs >= 256 ? pieces : std::max<int64_t>(4, (pieces * wgs + 255) / 256);
        span = std::max(span, (pieces + 255) / 256);      // 256 parts at most
        p.span = (int)std::min(span, pieces);
        p.splits = (int)((pieces + p.span - 1) / p.span);
        // With a prefix every tile leaves records, for the join to add the prefix's.
        p.records = p.splits == 1 && !a.pre.at ? 0 : (int)(wgs * p.splits);
    }
    p.acc = p.ml = nullptr;
    p.tickets = nullptr;
    return p;
}

size_t kv8_attend_workspace_bytes(const Kv8Attend &a) {
    const Kv8Plan p = kv8_plan(a);
    return (size_t)p.records * p.rows * (a.cache.D + 2) * sizeof(float);
}

template <int QT, int NH>
static hipError_t launch_kv8_decode_t(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    const size_t lds = std::max<size_t>(KVD_WAVES * 16 * (2 + a.cache.D + 4) * sizeof(float), 64 * KVD_WAVES * (sizeof(float4_t) + sizeof(float2_t)));
    static std::atomic<uint64_t> done{0};
    if (lds > 64 * 1024)
        if (hipError_t e = mx_allow_lds((const void *)kv8_attend_kernel<QT, NH>, (int)lds, done)) return e;
    hipLaunchKernelGGL((kv8_attend_kernel<QT, NH>), dim3((unsigned)p.wgs), dim3(64 * KVD_WAVES), lds, s, a, p);
    return hipGetLastError();
}

template <int QT>
static hipError_t launch_kv8_decode_q(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    switch ((a.cache.D + 63) / 64) {
        case 1: return launch_kv8_decode_t<QT, 1>(a, p, s);
        case 2: return launch_kv8_decode_t<QT, 2>(a, p, s);
        case 3: return launch_kv8_decode_t<QT, 3>(a, p, s);
        default: return launch_kv8_decode_t<QT, 4>(a, p, s);
    }
}

hipError_t launch_kv8_attend(const Kv8Attend &a, void *ws, hipStream_t s) {
    Kv8Plan p = kv8_plan(a);
    if (p.records) {
        p.acc = (float *)ws;
        p.ml = p.acc + (size_t)p.records * p.rows * a.cache.D;
        p.tickets = (uint32_t *)((char *)ws - COUNTER_BYTES);
    }
    if (p.rows == KVD_ROWS) return a.q_dt == DT_BF16 ? launch_kv8_decode_q<DT_BF16>(a, p, s) : launch_kv8_decode_q<DT_F16>(a, p, s);
    if (hipError_t e = launch_kv8_prefill(a, p, s); e != hipSuccess || !p.records) return e;
    const dim3 grid((unsigned)(p.tiles * (p.rows / KVJ_ROWS)), (unsigned)a.cache.H), block(KVJ_THREADS);
    const size_t lds = (size_t)KVJ_ROWS * p.splits * sizeof(float2_t);
    const bool bf16 = a.q_dt == DT_BF16;
    const auto join = a.pre.at ? (bf16 ? kv8_join_kernel<DT_BF16, true> : kv8_join_kernel<DT_F16, true>)
                               : (bf16 ? kv8_join_kernel<DT_BF16, false> : kv8_join_kernel<DT_F16, false>);
    hipLaunchKernelGGL(join, grid, block, lds, s, a, p);
    return hipGetLastError();
}

}  // namespace mcq4
