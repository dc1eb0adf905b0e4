// Attention of sequences that share a prefix: the rows of all of them (a row is a new token and one of a
// key/value head's G queries) go through the prefix's pages together, which so are read once for all; the sequences'
// own tokens are read by their rows alone.  Both are one kernel's work.  What a tile of rows makes of a stretch of
// tokens, unnormalised sums with their maximum and sum of weights, is left in a record, and a second kernel adds
// each row's records up.
//
// A prefix's rows, if they are many, take tiles of 128 through the core of the attention of prompts (kv8_prompt.h), a
// workgroup a tile.  Its sequences' own tokens, and prefixes of few rows, take tiles of 16, a wave a tile by itself:
// 64 tokens at a time from memory to registers, both products v_mfma_f32_16x16x32, as in kv8_attend.hip.  Scales, P in
// fp16 and the lag of a row's maximum are in both as in kv8_prompt.h: a row's largest weight stands at 2^7 to 2^15, so
// that weights below 2^-21 of it lose bits (each is off by 2^-31 of the largest at most) where kv8_attend.hip, with its
// largest at 2^15, keeps them down to 2^-29; most pieces leave the accumulators alone for that.  A CU holds workgroups
// of both kinds: the second are bound by memory, the first by neither it nor the matrix cores (below).
//
// Prefixes and contexts differ in length: the pieces of 64 tokens of all tiles of a kind stand in one row, by head, then
// prefixes, then sequences, and every workgroup (wave) takes an equal stretch of it.  Record t + w is that of stretch w's
// part of tile t: both rise along the row, so no two parts have one.  Stretches are numbered so that an XCD gets
// neighbouring ones, whose tiles read the same head's pages through one L2.
//
// Measured, 8 heads of keys, 4 queries each, D = 128, pages of 64 (both kernels; the first alone in brackets):
//   8 sequences of one token behind 2048 tokens, 1 to 162 of their own             15.8 us (13)    chains of loads: lengths,
//                                                                                  table, pieces; 5.7 MB
//   40 of three behind prefixes of 32768, 5000, 64 and 901, 3 to 1500 of their own 64 us (58)      0.32 PFLOP/s, 2.1 TB/s
//   64 of one behind 16384, 1 to 1024 of their own                                 52 us (48)      0.34 PFLOP/s, 2.0 TB/s
// The last two: the longest chains of a prefix's pieces (matrix cores and the VALU between their products) next to waves
// that wait for memory (VALU 37 to 40% busy, matrix cores 20%; 45% of the waves' time is waiting).  That is far from the same core
// in kv8_prefill.hip (35% and 47%): 128 rows a tile convert K and V twice as often, one operand is read ahead instead of four, and the
// instance of D = 128 takes all 256 registers, with 7 of them (32 bytes a lane) and 179 scalar ones spilled around the division
// of the work (D = 256: 28, 92 bytes, 264).  Tiles of 256 rows, a CU's eight waves
// for one, convert K and V half as often: 5 to 10% less where the prefix is all, 10 to 20% more beside long own contexts,
// whose waves then have CUs to themselves.  With tiles of 32 rows for the prefixes, whose pieces eight times as many workgroups read
// from L2, they took 138 and 119 us.
#include <algorithm>
#include <atomic>

#include "kv8_prompt.h"

namespace mcq4 {

constexpr int KVS_WAVES = 4, KVS_THREADS = 64 * KVS_WAVES;
constexpr int KVS_ROWS = KVP_WAVE_ROWS * KVS_WAVES, KVS_FEW = 16;      // rows of a tile of a workgroup, of a wave
// What a tile costs beside its pieces, in pieces: the chain of its lengths, table, codes and its record.
constexpr int KVS_START = 2, KVS_BIG_START = 2;
constexpr int kvs_k_buffers(int NT) { return NT <= 4 ? 2 : kvp_k_buffers(NT); }      // D <= 128: two workgroups a CU
// Operands read ahead: fewer than for prompts where registers are short.  D = 128, 256 a lane with two workgroups a CU:
// 40 sequences of 3 new tokens behind four prefixes (above) take 74.7 us with 4, 70 with 2, 67.5 with 1; a prefix of
// D = 256, 36.5 with 4 and 35.5 with 2.
constexpr int kvs_ahead(int NT) { return NT == 4 ? 1 : NT >= 7 ? 2 : kvp_ahead(NT); }
constexpr int kvs_lds(int NT) { return kvs_k_buffers(NT) * kvp_k_bytes(NT) + 2 * kvp_v_bytes(NT); }

// The rows of a prefix's sequences, or of a sequence, and the context that they go through.
struct Kv8Tiles {
    const int32_t *row;      // of the block table
    int width, ctx;
    int first, rows;         // first new token, rows of a key/value head
    int pos0;                // of new token 0 in the context; behind it where rows see all of it
    bool own;
};
template <int ROWS>
__device__ __forceinline__ int kvs_count(const Kv8Tiles &t) { return (t.rows + ROWS - 1) / ROWS; }
// Pieces of tile i, one where it sees none, so that its rows are written.
template <int ROWS>
__device__ __forceinline__ int kvs_pieces(const Kv8Attend &a, const Kv8Tiles &t, int i) {
    int end = t.ctx;
    if (t.own) {
        const int last = min((i + 1) * ROWS, t.rows) == t.rows ? t.rows / a.G - 1 : ((i + 1) * ROWS - 1) / a.G;
        end = min(max(t.pos0 + last + 1, 0), t.ctx);
    }
    return max(1, (end + KVD_STEP - 1) / KVD_STEP);
}

// Entry e of the list: prefixes, then sequences.
__device__ __forceinline__ Kv8Tiles kvs_tiles(const Kv8Attend &a, const Kv8Shared &x, int e) {
    const Kv8Batch &t = a.batch;
    Kv8Tiles o = {nullptr, 1, 0, 0, 0, 0, false};
    if (e < x.S) {
        int lo = 0, hi = t.B;
        if (x.groups) {
            lo = x.groups[e];
            hi = x.groups[e + 1];
            if (lo < 0 || hi < lo || hi > t.B) {
                o.rows = -1;
                return o;
            }
        } else if (x.S > 1) {
            const int each = t.B / x.S;
            lo = e * each;
            hi = lo + each;
        }
        const int from = t.cu ? t.cu[lo] : lo * t.each, to = t.cu ? t.cu[hi] : hi * t.each;
        if (from < 0 || to < from || to > t.T) {
            o.rows = -1;
            return o;
        }
        o.row = x.table + e * x.stride;
        o.width = x.W;
        o.ctx = min(max(x.lens[e], 0), x.W << a.cache.page_log);
        o.first = from;
        o.rows = (to - from) * a.G;
        o.pos0 = o.ctx;
    } else {
        const int b = e - x.S;
        const int from = t.cu ? t.cu[b] : b * t.each, to = t.cu ? t.cu[b + 1] : from + t.each;
        o.row = t.table + b * t.table_stride;
        o.width = t.W;
        o.ctx = min(max(t.lens[b], 0), t.W << a.cache.page_log);
        o.first = from;
        o.rows = ((from < 0) | (to < from) | (to > t.T)) ? -1 : (to - from) * a.G;
        o.pos0 = o.ctx - (to - from);
        o.own = true;
    }
    return o;
}
// The length of an entry's tiles in the row: their pieces, and START for each tile; 0xFFFFFFFF for offsets that are none.
template <int ROWS, int START>
__device__ __forceinline__ uint32_t kvs_length(const Kv8Attend &a, const Kv8Tiles &t) {
    const int n = kvs_count<ROWS>(t);
    if (n == 0) return t.rows < 0 ? 0xFFFFFFFFu : 0u;
    if (!t.own || n == 1) return (uint32_t)n * (uint32_t)(kvs_pieces<ROWS>(a, t, 0) + START);
    uint32_t sum = 0;
    for (int i = 0; i < n; ++i) sum += kvs_pieces<ROWS>(a, t, i) + START;
    return sum;
}

// A row of tiles of ROWS rows of entries [e0, e1), the same for every head, and where in it a wave stands.  Every lane takes part.
// Counts saturate: 0xFFFFFFFF is too many, as where an entry's offsets fall or leave their range.  Where none's do no token is two
// entries', and the records are enough.
template <int ROWS, int START>
struct Kv8Row {
    const Kv8Attend &a;
    const Kv8Shared &x;
    int e0;
    const int e1, lane;
    uint32_t length, tiles;                          // of a head
    struct Count { uint32_t length, tiles; } own, sum;
    int base;                                        // own and sum are of entries base .. base + 63,
    uint32_t before, tiles_before;                   // and these of those ahead of them

    static __device__ __forceinline__ uint32_t add(uint32_t p, uint32_t q) { return __builtin_elementwise_add_sat(p, q); }
    __device__ __forceinline__ uint32_t scan(uint32_t v) const {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d);
            if (lane >= d) v = add(v, up);
        }
        return v;
    }
    __device__ __forceinline__ Count count(int e) const {
        if (e >= e1) return {0, 0};
        const Kv8Tiles t = kvs_tiles(a, x, e);
        return {kvs_length<ROWS, START>(a, t), (uint32_t)kvs_count<ROWS>(t)};
    }
    __device__ __forceinline__ void block(int b) {
        base = b;
        own = count(b + lane);
        sum = {scan(own.length), scan(own.tiles)};
    }
    __device__ __forceinline__ Kv8Row(const Kv8Attend &a, const Kv8Shared &x, int e0, int e1)
        : a(a), x(x), e1(e1), lane(threadIdx.x & 63), before(0), tiles_before(0) { count_from(e0); }
    __device__ __forceinline__ void count_from(int first) {
        e0 = first;
        block(e0);
        length = own.length;
        tiles = own.tiles;
#pragma unroll 4
        for (int b = e0 + 64; b < e1; b += 64) {
            const Count n = count(b + lane);
            length = add(length, n.length);
            tiles = add(tiles, n.tiles);
        }
        length = e1 - e0 > 64 ? scan(length) : sum.length;
        tiles = e1 - e0 > 64 ? scan(tiles) : sum.tiles;
        length = __shfl(length, 63);
        tiles = __shfl(tiles, 63);
        length = kv8_same(length);
        tiles = kv8_same(tiles);
    }
    struct Tile {
        Kv8Tiles t;
        int e, i, pieces;
        uint32_t in, id;                             // place in the tile's length; number among the head's tiles
    };
    // Of place `at` < length, not ahead of the last one asked for (else `again`).
    __device__ __forceinline__ Tile find(uint32_t at, bool again) {
        if (again && base > e0) {
            before = tiles_before = 0;
            block(e0);
        }
        uint64_t past;
        while (!(past = __ballot(before + sum.length > at)) && base + 64 < e1) {
            before += __shfl(sum.length, 63);
            tiles_before += __shfl(sum.tiles, 63);
            block(base + 64);
        }
        const int k = past ? __builtin_ctzll(past) : 63;
        Tile o;
        o.e = base + k;
        o.t = kvs_tiles(a, x, o.e);
        o.t.ctx = kv8_same(o.t.ctx);
        o.t.first = kv8_same(o.t.first);
        o.t.rows = kv8_same(o.t.rows);
        o.t.pos0 = kv8_same(o.t.pos0);
        o.in = kv8_same(at - (before + __shfl(sum.length, k) - __shfl(own.length, k)));
        o.i = 0;
        o.pieces = kv8_same(kvs_pieces<ROWS>(a, o.t, 0));
        if (o.t.own) {                               // few tiles, of different lengths
            while (o.in >= (uint32_t)(o.pieces + START)) {
                o.in -= o.pieces + START;
                o.pieces = kvs_pieces<ROWS>(a, o.t, ++o.i);
            }
        } else if (o.in >= (uint32_t)(o.pieces + START)) {
            o.i = (int)(o.in / (uint32_t)(o.pieces + START));
            o.in -= (uint32_t)o.i * (o.pieces + START);
        }
        o.id = kv8_same(tiles_before + __shfl(sum.tiles, k) - __shfl(own.tiles, k) + o.i);
        return o;
    }
};

// Where the records of a tile's rows are: written by the part that begins it.
__device__ __forceinline__ void kvs_places(const Kv8Attend &a, const Kv8Tiles &t, int h, int r0, int rows, int2 *at, int record_row, int parts, int tid, int threads) {
    const int heads = a.cache.H * a.G;
    for (int rr = tid; rr < rows; rr += threads) {
        const int r = r0 + rr, tok = r / a.G;
        // A row that stands before its own context sees nothing, of its prefix either.
        at[(int64_t)(t.first + tok) * heads + h * a.G + (r - tok * a.G)] = int2{record_row + rr, !t.own || t.pos0 + tok >= 0 ? parts : 0};
    }
}

// A wave's 16 rows r0 .. of t through pieces c0 .. c1 - 1, to a record.
template <int QT, int NH>
__device__ __forceinline__ void kvs_few(const Kv8Attend &a, const Kv8Tiles &t, int h, int r0, int c0, int c1, float *acc_out, float *ml_out) {
    constexpr int ND = 4 * NH;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const Kv8Cache &c = a.cache;
    const int D = c.D, page_log = c.page_log, page = 1 << page_log;
    const int rows = min(KVS_FEW, t.rows - r0), r = r0 + min(col, rows - 1), tok = r / a.G;
    const int see = t.own ? min(t.pos0 + tok + 1, t.ctx) : t.ctx;

    const int k_sub = 16 * (col >> 2) + (col & 3);  // K row of token tile i: token k_sub + 4 i
    uint4_t kr[4][NH], vr[ND];
    int ek = 0, ev = 0, pv = -1;
    uint32_t kb = 0, vb = 0;
    auto pages = [&](int ci) {
        ek = t.row[min((ci * KVD_STEP + 16 * (col >> 2)) >> page_log, t.width - 1)];
        ev = t.row[min((ci * KVD_STEP + 16 * g) >> page_log, t.width - 1)];
    };
    auto fetch_k = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        const int pk = kv8_checked(ek, c.P, t0 + 16 * (col >> 2), t.ctx);
        pv = kv8_checked(ev, c.P, t0 + 16 * g, t.ctx);
        const int64_t bk = (int64_t)max(pk, 0) * c.H + h, bv = (int64_t)max(pv, 0) * c.H + h;
        kb = c.ks[bv];
        vb = c.vs[bv];
        const uint8_t *kp = c.k + bk * page * D + (int64_t)((t0 + k_sub) & (page - 1)) * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < NH; ++j) kr[i][j] = *(const uint4_t *)(kp + 4 * i * D + min(64 * j + 16 * g, D - 16));      // past D: q is 0
    };
    auto fetch_v = [&](int ci) {
        const int64_t bv = (int64_t)max(pv, 0) * c.H + h;
        const uint8_t *vp = c.v + bv * page * D + (int64_t)col * page + ((ci * KVD_STEP + 16 * g) & (page - 1));
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D) vr[i] = *(const uint4_t *)(vp + (int64_t)16 * i * page);
    };
    pages(c0);
    // A negative scale goes into q's sign, so that the scores' factor is positive.
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    const uint16_t *q = (const uint16_t *)a.q + (int64_t)(t.first + tok) * a.q_token + (int64_t)(h * a.G + (r - tok * a.G)) * a.q_head;
    uint4_t qv[NH][2];
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int d = 64 * j + 16 * g + 8 * u;
            qv[j][u] = d < D ? *(const uint4_t *)(q + d) : uint4_t{0, 0, 0, 0};
        }
    fetch_k(c0);
    fetch_v(c0);
    pages(c0 + 1);
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) qv[j][u][e] ^= flip;

    float4_t acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    float m = -__FLT_MAX__, l = 0.f;                 // m is finite from the start: no score needs a case of its own
    int rest = KVP_P_LOG - (int)KV8_NO_K;            // KVP_P_LOG - k
    const float qk = fabsf(a.scale) * LOG2E;

    for (int ci = c0; ci < c1; ++ci) {
        const bool more = ci + 1 < c1;
        // Of the lane's 16 tokens the row sees the first `seen`.
        const bool here = pv >= 0;
        const int seen = here ? min(max(see - (ci * KVD_STEP + 16 * g), 0), 16) : 0;
        const bool full = __all(seen == 16);
        // Never 0 (masked scores are -inf); NaN only where its page has tokens that are seen.
        const float f = kb == 255 && seen > 0 ? NAN : fmaxf(qk * __uint_as_float((kb < 255 ? kb : 0u) << 23), 0x1p-126f);
        const bool v_nan = here && vb == 255;
        const int vbyte = here ? (int)vb : 0;
        float4_t s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NH; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) s[i] = mx_mfma16<QT>(kv8_eight<QT>(kr[i][j][2 * u], kr[i][j][2 * u + 1], 1.0f), qv[j][u], s[i]);
        }
        if (more) fetch_k(ci + 1);
        if (!full)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][e] = 4 * i + e < seen ? s[i][e] : -INFINITY;
        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[i][e]);
        mx *= f;
        const float top = kv8_group_max(mx);
        const bool moved = top > m + KVP_LAG;
        if (__any(moved | (rest > KVP_P_LOG + KVP_V_LAG - vbyte))) {
            const float m_new = moved ? top : m, drop = m - m_new;
            const float most = kv8_group_max(mx - m_new + (float)vbyte) + kvp_room(m_new);
            const bool over = moved | (most + (float)rest > 15.f);      // of this row: others' do not change its k
            if (__any(over)) {
                m = m_new;
                l *= __builtin_amdgcn_exp2f(drop);
                const float before = (float)rest;
                rest = over ? KVP_P_LOG - (int)ceilf(kv8_k(fmaxf(KVP_P_LOG - before + drop, most))) : rest;
                const float shrink = __builtin_amdgcn_exp2f(drop + ((float)rest - before));
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[i] *= shrink;
            }
        }
        const int log = max(rest + vbyte, (int)KV8_LEAST);
        const float b = (float)log - m;
        float add = 0.f;
        uint4_t pr[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], f, b));
                add += s[i][e];
            }
            pr[i >> 1][2 * (i & 1)] = bitcast<uint32_t>(half2_t{(_Float16)s[i][0], (_Float16)s[i][1]});
            pr[i >> 1][2 * (i & 1) + 1] = bitcast<uint32_t>(half2_t{(_Float16)s[i][2], (_Float16)s[i][3]});
        }
        l += __builtin_ldexpf(add, -log);
        if (__any(v_nan)) {                          // byte 255: every value of the page
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
                    for (int e = 0; e < 4; ++e) {
                        vr[i][e] = here ? vr[i][e] : 0u;
                        bad |= kv8_nan_bytes(vr[i][e]);
                    }
        }
        if (__any(bad != 0)) {
            // NaN of V where not every row sees every token: counted for each row and channel by a product of ones, and taken out.
            uint4_t pn[2];
#pragma unroll
            for (int e = 0; e < 16; e += 2) pn[e >> 3][(e >> 1) & 3] = (e < seen ? 0x3C00u : 0u) | (e + 1 < seen ? 0x3C000000u : 0u);
#pragma unroll
            for (int i = 0; i < ND; ++i)
                if (16 * i < D) {
                    uint4_t n;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w = kv8_nan_bytes(vr[i][e]);
                        n[e] = w & 0x38383838u;                       // e4m3's 1.0
                        vr[i][e] &= ~w;
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
                for (int u = 0; u < 2; ++u) acc[i] = mx_mfma16<DT_F16>(kv8_eight<DT_F16>(vr[i][2 * u], vr[i][2 * u + 1], 1.0f), pr[u], acc[i]);
        if (more) {
            fetch_v(ci + 1);
            pages(ci + 2);
        }
    }
    l = kv8_group_sum(l);
    if (col >= rows) return;
    const int unit = -rest - 127;                    // the accumulators' exponent
#pragma unroll
    for (int i = 0; i < ND; ++i)
        if (16 * i < D)
            *(float4_t *)(acc_out + col * D + 16 * i + 4 * g) = float4_t{__builtin_ldexpf(acc[i][0], unit), __builtin_ldexpf(acc[i][1], unit),
                                                                         __builtin_ldexpf(acc[i][2], unit), __builtin_ldexpf(acc[i][3], unit)};
    if (g == 0) *(float2_t *)(ml_out + 2 * col) = float2_t{m, l};
}

// MANY: prefixes in tiles of 128 rows (else of 16).  own: the sequences' own tokens too.
template <int QT, int NT, bool MANY>
__global__ void __launch_bounds__(KVS_THREADS, NT <= 4 ? 2 : 1)
kv8_shared_kernel(Kv8Attend a, Kv8Shared x, int own) {
    const int tid = threadIdx.x, lane = tid & 63, H = a.cache.H, heads = H * a.G, D = a.cache.D;
    const uint32_t wgs = gridDim.x;
    const Kv8Batch &t = a.batch;
    // Tokens of no prefix, and of no sequence, have no records.
    if (x.groups && (x.groups[0] != 0 || x.groups[x.S] != t.B)) {
        const int lo = min(max(x.groups[0], 0), t.B), hi = min(max(x.groups[x.S], 0), t.B);
        const int t0 = t.cu ? t.cu[lo] : lo * t.each, t1 = t.cu ? t.cu[hi] : hi * t.each;
        for (int k = blockIdx.x; k < t.T; k += wgs)
            if (k < t0 || k >= t1)
                for (int r = tid; r < heads; r += KVS_THREADS) a.pre.at[(int64_t)k * heads + r] = int2{0, 0};
    }
    if (t.cu && (t.cu[0] != 0 || t.cu[t.B] != t.T))
        for (int k = blockIdx.x; k < t.T; k += wgs)
            if (k < t.cu[0] || k >= t.cu[t.B])
                for (int r = tid; r < heads; r += KVS_THREADS) (own ? a.pre.own_at : a.pre.at)[(int64_t)k * heads + r] = int2{0, 0};

    const uint32_t most = 0x7FFFFFFFu / (uint32_t)H;
    Kv8Row<KVS_ROWS, KVS_BIG_START> big(a, x, 0, MANY ? x.S : 0);
    Kv8Row<KVS_FEW, KVS_START> few(a, x, MANY ? x.S : 0, x.S + (own ? t.B : 0));
    // Offsets that fall or leave their range, as every workgroup finds: of groups, and no sequence has a prefix; of new tokens, and no
    // row is a sequence's.  The rows say that they have no records, so that nothing of an earlier call's is added to them.  (Out of
    // the way of the others: a loop around both counts has all arguments fetched ahead of it, one after another, 0.7 us.)
    bool no_own = few.length > most || (int64_t)few.tiles * H + KVS_WAVES * wgs > a.pre.own_records, no_prefix = no_own;
    if constexpr (MANY) no_prefix = big.length > most || (int64_t)big.tiles * H + wgs > a.pre.records;
    if (__builtin_expect(no_prefix | no_own, 0)) {
        if constexpr (!MANY) {
            few.count_from(x.S);
            no_own = few.length > most || (int64_t)few.tiles * H + KVS_WAVES * wgs > a.pre.own_records;
        }
        for (int64_t r = (int64_t)blockIdx.x * KVS_THREADS + tid; r < (int64_t)t.T * heads; r += (int64_t)wgs * KVS_THREADS) {
            if (no_prefix) a.pre.at[r] = int2{0, 0};
            if (no_own) a.pre.own_at[r] = int2{0, 0};
        }
        if (no_own) return;
    }
    const uint32_t big_length = MANY && !no_prefix ? big.length : 0;
    // How many of the workgroups take tiles of 128 rows, of each XCD's as many.
    const uint32_t parts8 = wgs % 8 ? 1 : 8, local = wgs / parts8, mine = blockIdx.x / parts8, xcd = blockIdx.x % parts8;
    const uint64_t cost_big = (uint64_t)big_length * a.pre.cost, cost_few = few.length;
    uint32_t local_big = 0;
    if (big_length) local_big = few.length ? (uint32_t)min((uint64_t)local - 1, max((uint64_t)1, (local * cost_big + (cost_big + cost_few) / 2) / (cost_big + cost_few))) : local;
    if constexpr (MANY)
    if (mine < local_big) {
        extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
        // An XCD's stretch of the row, and its workgroups': those that come first to its 32 CUs take 8 pieces where those that come
        // second to one, which the first one's waves delay, take 7 (the prefix of 16384 tokens: 53.9 us with equal parts, 52.2).
        const uint32_t all = big.length * H, each = (all + parts8 - 1) / parts8, firsts = min(local_big, 32u), seconds = local_big - firsts;
        const uint32_t shares = 8 * firsts + 7 * seconds;
        const uint32_t chunk1 = max(each / shares * 8 + (each % shares * 8 + shares - 1) / shares, (uint32_t)(KVS_BIG_START + 1));
        const uint32_t front = min(firsts * chunk1, each), chunk2 = max((each - front + max(seconds, 1u) - 1) / max(seconds, 1u), (uint32_t)(KVS_BIG_START + 1));
        auto place = [&](uint32_t in) { return in < front ? in / chunk1 : firsts + (in - front) / chunk2; };
        const uint32_t used = place(each - 1) + 1, w = xcd * used + mine;       // none without a part among them
        const uint32_t stop = min((xcd + 1) * each, all), start = min(xcd * each + (mine < firsts ? mine * chunk1 : front + (mine - firsts) * chunk2), stop);
        const uint32_t end = mine < used ? min(start + (mine < firsts ? chunk1 : chunk2), stop) : start;
        auto part = [&](uint32_t at) { return at / each * used + place(at % each); };
        const Kv8Batch tb = {x.table, x.stride, x.S, x.W, x.lens, nullptr, 0, 0};
        int h = (int)(start / big.length);
        uint32_t in_head = start - h * big.length;
        bool again = false;
        for (uint32_t at = start; at < end;) {
            const auto o = big.find(in_head, again);
            again = false;
            // A tile's length: its start, then its pieces.
            const uint32_t n1 = min((uint32_t)(o.pieces + KVS_BIG_START) - o.in, end - at), first = at - o.in + KVS_BIG_START;
            const int c0 = max((int)o.in - KVS_BIG_START, 0), c1 = (int)(o.in + n1) - KVS_BIG_START;
            const uint32_t tile = h * big.tiles + o.id;
            const int r0 = o.i * KVS_ROWS, rows = min(KVS_ROWS, o.t.rows - r0);
            at += n1;
            in_head += n1;
            const int head = h;
            if (in_head == big.length) {
                in_head = 0;
                again = true;
                ++h;
            }
            if (c1 <= c0) continue;
            if (c0 == 0) {
                const uint32_t begun = part(first);
                kvs_places(a, o.t, head, r0, rows, a.pre.at, (int)(tile + begun) * KVS_ROWS, (int)(part(first + o.pieces - 1) - begun + 1), tid, KVS_THREADS);
            }
            const int64_t record = (int64_t)(tile + w) * KVS_ROWS;
            const Kv8Rows R = {o.e, r0, o.t.rows, o.t.first, o.t.ctx, o.t.ctx, 0, o.pieces};
            kvp_attend<QT, NT, KVS_WAVES, kvs_k_buffers(NT), kvs_ahead(NT)>(a, tb, 0, 0, R, head, c0, c1, smem,
                                                             [&](int row, int hi, const float16_t (&acc)[NT], int unit, float m, float l) {
                if (row >= rows) return;
                float *const out = a.pre.acc + (record + row) * D + 4 * hi;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (32 * i + 8 * e < D)
                            *(float4_t *)(out + 32 * i + 8 * e) = float4_t{__builtin_ldexpf(acc[i][4 * e], unit), __builtin_ldexpf(acc[i][4 * e + 1], unit),
                                                                           __builtin_ldexpf(acc[i][4 * e + 2], unit), __builtin_ldexpf(acc[i][4 * e + 3], unit)};
                if (hi == 0) *(float2_t *)(a.pre.ml + (record + row) * 2) = float2_t{m, l};
            });
            __syncthreads();                         // LDS has been read
            if (at < end) big.block(big.base);       // counted again: no registers over the tile for it
        }
        return;
    }
    if (!few.length) return;
    const uint32_t local_few = local - local_big, n = local_few * parts8 * KVS_WAVES;
    const uint32_t w = (xcd * local_few + mine - local_big) * KVS_WAVES + __builtin_amdgcn_readfirstlane(tid >> 6), all = few.length * H;
    const uint32_t chunk = max((all + n - 1) / n, (uint32_t)(KVS_START + 1));
    const uint32_t start = (uint32_t)min((uint64_t)w * chunk, (uint64_t)all), end = min(start + chunk, all);
    int h = (int)(start / few.length);
    uint32_t in_head = start - h * few.length;
    bool again = false;
    for (uint32_t at = start; at < end;) {
        const auto o = few.find(in_head, again);
        again = false;
        // A tile's length: KVS_START, then its pieces.
        const uint32_t n1 = min((uint32_t)(o.pieces + KVS_START) - o.in, end - at), first = at - o.in + KVS_START, begun = first / chunk;
        const int c0 = max((int)o.in - KVS_START, 0), c1 = (int)(o.in + n1) - KVS_START;
        if (c1 > c0) {
            const uint32_t tile = h * few.tiles + o.id;
            const int r0 = o.i * KVS_FEW, rows = min(KVS_FEW, o.t.rows - r0);
            const int rec_rows = o.t.own ? a.pre.own_rows : KVS_FEW;
            if (c0 == 0)
                kvs_places(a, o.t, h, r0, rows, o.t.own ? a.pre.own_at : a.pre.at, (int)(tile + begun) * rec_rows,
                           (int)((first + o.pieces - 1) / chunk - begun + 1), lane, 64);
            const int64_t record = (int64_t)(tile + w) * rec_rows;
            kvs_few<QT, (NT + 1) / 2>(a, o.t, h, r0, c0, c1, (o.t.own ? a.pre.own_acc : a.pre.acc) + record * D,
                                      (o.t.own ? a.pre.own_ml : a.pre.ml) + record * 2);
        }
        at += n1;
        in_head += n1;
        if (in_head == few.length) {
            in_head = 0;
            again = true;
            ++h;
        }
    }
}

// The rows' records added up, their own tokens' and then the prefix's: a thread takes four channels of a row and every
// fourth part, and the four threads' sums are added in LDS (one thread for all parts: 8.5 us where it is 6.9,
// and 5.6 for 4.2; the prefix's parts in a loop behind the others': 10.3 for 7.8).
constexpr int KVSJ_BATCH = 8, KVSJ_GROUPS = 4, KVSJ_UNITS = 64;
template <int QT>
__global__ void __launch_bounds__(KVSJ_GROUPS * KVSJ_UNITS)
kv8_shared_join_kernel(Kv8Attend a) {
    __shared__ __attribute__((aligned(16))) float4_t gacc[KVSJ_GROUPS][KVSJ_UNITS];
    __shared__ __attribute__((aligned(8))) float2_t gml[KVSJ_GROUPS][KVSJ_UNITS];
    const int D = a.cache.D, D4 = D >> 2, each = KVSJ_UNITS / D4, u = threadIdx.x % KVSJ_UNITS, g = threadIdx.x / KVSJ_UNITS;
    const int64_t rows = (int64_t)a.batch.T * a.cache.H * a.G, o = (int64_t)blockIdx.x * each + u / D4;
    const int d = 4 * (u % D4);
    const bool on = u < each * D4 && o < rows;
    float top = -INFINITY, l = 0.f;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    if (on) {
        const int2 own = a.pre.own_at[o], pre = a.pre.at[o];
        // Parts that would not lie among the records (of rows of groups that fall) are none.
        auto parts = [](int2 at, int rows, int64_t records) { return at.y > 0 && at.x >= 0 && at.x + (int64_t)(at.y - 1) * rows < records * rows ? at.y : 0; };
        const int n0 = parts(own, a.pre.own_rows, a.pre.own_records), n1 = own.y > 0 ? parts(pre, a.pre.rows, a.pre.records) : 0;
        for (int s0 = g; s0 < n0 + n1; s0 += KVSJ_GROUPS * KVSJ_BATCH) {
            float2_t ml[KVSJ_BATCH];
            float4_t x[KVSJ_BATCH];
#pragma unroll
            for (int i = 0; i < KVSJ_BATCH; ++i) {
                const int s = s0 + i * KVSJ_GROUPS;
                ml[i] = float2_t{-INFINITY, 0.f};
                x[i] = float4_t{0.f, 0.f, 0.f, 0.f};
                if (s < n0 + n1) {
                    const bool p = s >= n0;
                    const int64_t row = p ? pre.x + (int64_t)(s - n0) * a.pre.rows : own.x + (int64_t)s * a.pre.own_rows;
                    ml[i] = *(const float2_t *)((p ? a.pre.ml : a.pre.own_ml) + row * 2);
                    x[i] = *(const float4_t *)((p ? a.pre.acc : a.pre.own_acc) + row * D + d);
                }
            }
            float most = top;
#pragma unroll
            for (int i = 0; i < KVSJ_BATCH; ++i) most = fmaxf(most, ml[i][0]);
            const float use = most == -INFINITY ? 0.f : most, shrink = __builtin_amdgcn_exp2f(top - use);
            top = most;
            l *= shrink;
            v *= shrink;
#pragma unroll
            for (int i = 0; i < KVSJ_BATCH; ++i) {
                const float w = __builtin_amdgcn_exp2f(ml[i][0] - use);
                l += ml[i][1] * w;
                v += x[i] * w;
            }
        }
    }
    gacc[g][u] = v;
    gml[g][u] = float2_t{top, l};
    __syncthreads();
    if (g || !on) return;
#pragma unroll
    for (int i = 1; i < KVSJ_GROUPS; ++i) top = fmaxf(top, gml[i][u][0]);
    const float use = top == -INFINITY ? 0.f : top, w0 = __builtin_amdgcn_exp2f(gml[0][u][0] - use);
    l *= w0;
    v *= w0;
#pragma unroll
    for (int i = 1; i < KVSJ_GROUPS; ++i) {
        const float w = __builtin_amdgcn_exp2f(gml[i][u][0] - use);
        l += gml[i][u][1] * w;
        v += gacc[i][u] * w;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;            // a row that sees nothing is 0
    *(uint2_t *)((uint16_t *)a.out + o * D + d) = uint2_t{mx_pair<QT>(v[0] * inv, v[1] * inv), mx_pair<QT>(v[2] * inv, v[3] * inv)};
    if (a.lse && d == 0) a.lse[o] = l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * (1.0f / LOG2E);
}

namespace {
struct Plan {
    bool many, own;               // prefixes in tiles of 128 rows; the sequences' own tokens too
    int wgs, own_rows, rows;
    int64_t records, own_records;
};
Plan shared_plan(const Kv8Attend &a, const Kv8Shared &x) {
    Plan p;
    const Kv8Batch &b = a.batch;
    const int64_t rows = (int64_t)b.T * a.G, step = (int64_t)1 << a.cache.page_log;
    auto pieces = [&](int64_t width, int64_t most) { return std::max<int64_t>(1, (std::min(width * step, most) + KVD_STEP - 1) / KVD_STEP); };
    // Many new tokens each: tiles of 16 rows read a sequence's context again and again.  Four queries a token, bf16, with them and
    // with the prompts' kernels: D = 128, 64 rows of 8192 of its own 56 and 76 us, 128 rows 87 and 83, of 4096 164 and 120;
    // D = 64, 128 rows of 8192 50 and 65, 192 rows of 4096 123 and 114; D = 256, 64 rows of 4096 110 and 115, 128 rows 208 and 132.
    // By the call's average: one long prompt among single tokens takes tiles of 16 rows too, which read its own context again for
    // each (200 single tokens and a prompt of 3000, behind 2048: 863 us, while calls of their own would take 57 and 315; 63 and one
    // of 512: 127, and 27 and 97).
    p.own = rows / b.B <= (a.cache.D <= 64 ? 128 : 80);
    if (const char *v = opt("MCQ4_KV8_ROWS")) p.own = atoi(v) <= KVD_ROWS;
    // Their pieces, and those of prefixes (2^30 at most) beside them, are counted in 31 bits, whatever the contexts turn out to be.
    const int64_t own_tiles = rows / KVS_FEW + b.B;
    if ((b.W * step / KVD_STEP + 2 + KVS_START) * own_tiles > ((int64_t)1 << 29) / a.cache.H) p.own = false;
    // Rows of a prefix, four of 16384 tokens each, in tiles of 16 and of 128: D = 128, 32 rows 53.4 and 51.7 us, 40 rows 73 and 58;
    // D = 64, where a CU holds more waves, 64 rows 46.2 and 46.9, 96 rows 67 and 52; D = 256, where a CU holds one workgroup of the
    // large tiles, 48 rows 77.0 and 77.7, 96 rows 137 and 89.
    p.many = rows / x.S > (a.cache.D > 64 && a.cache.D <= 128 ? 32 : 64) || !p.own;
    if (const char *v = opt("MCQ4_KV8_PREFIX_ROWS")) p.many = atoi(v) > KVS_FEW || !p.own;
    p.rows = p.many ? KVS_ROWS : KVS_FEW;
    const int64_t prefix_tiles = rows / p.rows + x.S;
    const int64_t big = p.many ? prefix_tiles * (pieces(x.W, x.max_prefix) + KVS_BIG_START) : 0;
    const int64_t few = (p.many ? 0 : prefix_tiles * (pieces(x.W, x.max_prefix) + KVS_START)) + (p.own ? own_tiles * (pieces(b.W, a.max_context) + KVS_START) : 0);
    // As many workgroups as the CUs hold at once: two each, or one where D > 128 takes the registers.
    p.wgs = (int)std::min<int64_t>(a.cache.D <= 128 ? 512 : 256, (big / (KVS_BIG_START + 1) + few / (KVS_WAVES * (KVS_START + 1)) + 2) * a.cache.H);
    if (const char *v = opt("MCQ4_KV8_PREFIX_WGS")) p.wgs = std::max(1, std::min(2048, atoi(v)));
    if (p.many && p.own) p.wgs = std::max(p.wgs, 16);        // some of each kind, on every XCD
    if (p.wgs > 8) p.wgs = (p.wgs + 7) / 8 * 8;
    p.own_rows = b.cu ? KVS_FEW : (int)std::min<int64_t>(KVS_FEW, (int64_t)b.each * a.G);
    p.records = prefix_tiles * a.cache.H + p.wgs * (p.many ? 1 : KVS_WAVES);
    p.own_records = (own_tiles + (p.many ? 0 : prefix_tiles)) * a.cache.H + p.wgs * KVS_WAVES;
    if (!p.many) p.records = p.own_records;                  // numbered together
    return p;
}
}  // namespace

bool kv8_shared_own(const Kv8Attend &a, const Kv8Shared &x) { return shared_plan(a, x).own; }

size_t kv8_shared_bytes(const Kv8Attend &a, const Kv8Shared &x, Kv8Prefix *out, void *ws) {
    const Plan p = shared_plan(a, x);
    char *at = (char *)ws;
    auto take = [&](size_t n) {
        char *const here = at;
        at += (n + 15) / 16 * 16;
        return here;
    };
    const size_t rows = (size_t)a.batch.T * a.cache.H * a.G, D = a.cache.D;
    *out = {};
    out->records = p.records;
    out->own_records = p.own_records;
    out->rows = p.rows;
    out->own_rows = p.own_rows;
    out->cost = 4;       // with 3 the four prefixes take 67.5 us (4: 65.5), the one of 16384 tokens 52.7 (52.1)
    if (const char *v = opt("MCQ4_KV8_PREFIX_COST")) out->cost = std::max(1, std::min(64, atoi(v)));
    out->at = (int2 *)take(rows * sizeof(int2));
    out->acc = (float *)take(p.records * p.rows * D * sizeof(float));
    out->ml = (float *)take(p.records * p.rows * 2 * sizeof(float));
    if (p.own) {
        out->own_at = (int2 *)take(rows * sizeof(int2));
        out->own_acc = (float *)take(p.own_records * p.own_rows * D * sizeof(float));
        out->own_ml = (float *)take(p.own_records * p.own_rows * 2 * sizeof(float));
    }
    return at - (char *)ws;
}

template <int QT, int NT>
static hipError_t launch_kv8_shared_t(const Kv8Attend &a, const Kv8Shared &x, const Plan &p, hipStream_t s) {
    constexpr int lds = kvs_lds(NT);
    static_assert(lds + 16 * kvp_channels(NT) + 64 <= (NT <= 4 ? 80 : 160) * 1024, "LDS budget");
    if (p.many) {
        static std::atomic<uint64_t> done{0};
        if (lds > 64 * 1024)
            if (hipError_t e = mx_allow_lds((const void *)kv8_shared_kernel<QT, NT, true>, lds, done)) return e;
        hipLaunchKernelGGL((kv8_shared_kernel<QT, NT, true>), dim3((unsigned)p.wgs), dim3(KVS_THREADS), lds, s, a, x, (int)p.own);
    } else {
        hipLaunchKernelGGL((kv8_shared_kernel<QT, NT, false>), dim3((unsigned)p.wgs), dim3(KVS_THREADS), 0, s, a, x, (int)p.own);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (!p.own) return hipSuccess;
    const int64_t rows = (int64_t)a.batch.T * a.cache.H * a.G, each = KVSJ_UNITS / (a.cache.D >> 2);
    hipLaunchKernelGGL(kv8_shared_join_kernel<QT>, dim3((unsigned)((rows + each - 1) / each)), dim3(KVSJ_GROUPS * KVSJ_UNITS), 0, s, a);
    return hipGetLastError();
}
template <int QT>
static hipError_t launch_kv8_shared_q(const Kv8Attend &a, const Kv8Shared &x, hipStream_t s) {
    const Plan p = shared_plan(a, x);
    switch ((a.cache.D + 31) / 32) {
        case 1: return launch_kv8_shared_t<QT, 1>(a, x, p, s);
        case 2: return launch_kv8_shared_t<QT, 2>(a, x, p, s);
        case 3: return launch_kv8_shared_t<QT, 3>(a, x, p, s);
        case 4: return launch_kv8_shared_t<QT, 4>(a, x, p, s);
        case 5: return launch_kv8_shared_t<QT, 5>(a, x, p, s);
        case 6: return launch_kv8_shared_t<QT, 6>(a, x, p, s);
        case 7: return launch_kv8_shared_t<QT, 7>(a, x, p, s);
        default: return launch_kv8_shared_t<QT, 8>(a, x, p, s);
    }
}
hipError_t launch_kv8_shared(const Kv8Attend &a, const Kv8Shared &x, hipStream_t s) {
    return a.q_dt == DT_BF16 ? launch_kv8_shared_q<DT_BF16>(a, x, s) : launch_kv8_shared_q<DT_F16>(a, x, s);
}

}  // namespace mcq4
