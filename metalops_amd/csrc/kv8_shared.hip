// Attention of sequences that share a prefix: the rows of all of them (a row is a new token and one of a
// key/value head's G queries) go through the prefix's pages together, which so are read once for all.  What
// they make of it, unnormalised sums with their maximum and sum of weights, is left in records; the kernels of
// the sequences' own tokens (kv8_attend.hip) add those of a row when they write it.
//
// Operands are as in kv8_attend.hip: a wave takes 64 tokens at a time from memory to registers, turns
// codes into 16 bits there, and both products are v_mfma_f32_16x16x32 with the cache as the A operand, but for
// RT tiles of 16 rows at once, so that a code is read and converted once for 16 RT rows.  Scales, P in fp16
// and the lag of a row's maximum are those of kv8_prefill.hip.  Every row sees the same tokens, so masks are of
// the prefix's end and of pages that are not there, and V's codes behind it are taken as 0.
//
// Prefixes differ in length and in their rows: as in kv8_attend.hip the pieces of 64 tokens of all tiles stand
// in one row, by head, prefix, tile and token, and every workgroup takes an equal stretch of it.  Record r + w
// is that of stretch w's part of tile r: both rise along the row, so no two parts have one.  Stretches are
// numbered so that an XCD gets neighbouring ones, whose tiles read the same head's pages through one L2.
#include <algorithm>
#include <atomic>

#include "kv8_attend.h"

namespace mcq4 {

constexpr int KVS_WAVES = 4;
constexpr int KVS_LAG = 7, KVS_V_LAG = 1, KVS_P_LOG = 15 - KVS_LAG - KVS_V_LAG;

struct Kv8Group { int first, rows, ctx, tiles, pieces; };      // first token, rows of a key/value head; pieces of a tile
template <int ROWS>
__device__ __forceinline__ Kv8Group kv8_group(const Kv8Attend &a, const Kv8Shared &x, int s) {
    const Kv8Batch &t = a.batch;
    Kv8Group g = {0, 0, 0, 0, 1};
    const int each = t.B / x.S, lo = x.groups ? x.groups[s] : s * each, hi = x.groups ? x.groups[s + 1] : lo + each;
    if (lo < 0 || hi < lo || hi > t.B) return g;
    const int from = t.cu ? t.cu[lo] : lo * t.each, to = t.cu ? t.cu[hi] : hi * t.each;
    if (from < 0 || to < from || to > t.T) return g;
    g.first = from;
    g.rows = (to - from) * a.G;
    g.tiles = (g.rows + ROWS - 1) / ROWS;
    g.ctx = min(max(x.lens[s], 0), x.W << a.cache.page_log);
    g.pieces = max(1, (g.ctx + KVD_STEP - 1) / KVD_STEP);
    return g;
}

struct Kv8Part { int s, h, r0, c0, c1, record; };

// A wave's part of a tile: RT times 16 rows, pieces c0 + wave, c0 + wave + 4, ..; then the four waves' sums to the record.
template <int QT, int NH, int RT>
__device__ __forceinline__ void kv8_prefix_tile(const Kv8Attend &a, const Kv8Shared &x, const Kv8Group &G, const Kv8Part &w, uint8_t *smem) {
    constexpr int ND = 4 * NH, ROWS = 16 * RT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const Kv8Cache &c = a.cache;
    const int D = c.D, page_log = c.page_log, page = 1 << page_log, ctx = G.ctx;
    const Kv8Batch table = {x.table, x.stride, x.S, x.W, x.lens, nullptr, 0, 0};

    // A negative scale goes into q's sign, so that the scores' factor is positive.
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    uint4_t qv[RT][NH][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(w.r0 + 16 * rt + col, G.rows - 1);
        const uint16_t *q = (const uint16_t *)a.q + (int64_t)(G.first + r / a.G) * a.q_token + (int64_t)(w.h * a.G + r % a.G) * a.q_head;
#pragma unroll
        for (int i = 0; i < NH; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 64 * i + 16 * g + 8 * u;
                qv[rt][i][u] = d < D ? *(const uint4_t *)(q + d) : uint4_t{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; ++e) qv[rt][i][u][e] ^= flip;
            }
    }
    float4_t acc[RT][ND];
    float m[RT], l[RT];                              // m is finite from the start: no score needs a case of its own
    int rest[RT];                                    // KVS_P_LOG - k
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__FLT_MAX__;
        l[rt] = 0.f;
        rest[rt] = KVS_P_LOG - (int)KV8_NO_K;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[rt][i] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const float qk = fabsf(a.scale) * LOG2E;

    const int k_sub = 16 * (col >> 2) + (col & 3);  // K row of tile t: token k_sub + 4 t
    uint4_t kr[4][NH], vr[ND];
    int ek = 0, ev = 0, pv = -1;
    uint32_t kb = 0, vb = 0;
    auto pages = [&](int ci) {
        ek = kv8_entry(table, page_log, w.s, ci * KVD_STEP + 16 * (col >> 2));
        ev = kv8_entry(table, page_log, w.s, ci * KVD_STEP + 16 * g);
    };
    auto fetch_k = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        const int pk = kv8_checked(ek, c.P, t0 + 16 * (col >> 2), ctx);
        pv = kv8_checked(ev, c.P, t0 + 16 * g, ctx);
        const int64_t bk = (int64_t)max(pk, 0) * c.H + w.h, bv = (int64_t)max(pv, 0) * c.H + w.h;
        kb = c.ks[bv];
        vb = c.vs[bv];
        const uint8_t *kp = c.k + bk * page * D + (int64_t)((t0 + k_sub) & (page - 1)) * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < NH; ++i) kr[t][i] = *(const uint4_t *)(kp + 4 * t * D + min(64 * i + 16 * g, D - 16));      // past D: q is 0
    };
    auto fetch_v = [&](int ci) {
        const int64_t bv = (int64_t)max(pv, 0) * c.H + w.h;
        const uint8_t *vp = c.v + bv * page * D + (int64_t)col * page + ((ci * KVD_STEP + 16 * g) & (page - 1));
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D) vr[i] = *(const uint4_t *)(vp + (int64_t)16 * i * page);
    };

    if (w.c0 + wave < w.c1) {
        pages(w.c0 + wave);
        fetch_k(w.c0 + wave);
        fetch_v(w.c0 + wave);
        pages(w.c0 + wave + KVS_WAVES);
    }
    for (int ci = w.c0 + wave; ci < w.c1; ci += KVS_WAVES) {
        const bool more = ci + KVS_WAVES < w.c1;
        const int t_own = ci * KVD_STEP + 16 * g;
        // Of the lane's 16 tokens as many are seen, by every row.
        const int seen = pv >= 0 ? min(ctx - t_own, 16) : 0;
        const bool full = __all(seen == 16);
        const float f = kb == 255 ? NAN : fmaxf(qk * __uint_as_float(kb << 23), 0x1p-126f);      // never 0: masked scores are -inf
        const bool v_nan = seen > 0 && vb == 255;
        const int vbyte = seen > 0 ? (int)vb : 0;
        float4_t s[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            uint4_t op[NH][2];
#pragma unroll
            for (int i = 0; i < NH; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u) op[i][u] = kv8_eight<QT>(kr[t][i][2 * u], kr[t][i][2 * u + 1], 1.0f);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s[rt][t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NH; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) s[rt][t] = mx_mfma16<QT>(op[i][u], qv[rt][i][u], s[rt][t]);
            }
        }
        if (more) fetch_k(ci + KVS_WAVES);
        uint4_t pr[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (!full)
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[rt][t][i] = 4 * t + i < seen ? s[rt][t][i] : -INFINITY;
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][t][i]);
            mx = seen > 0 ? mx * f : -INFINITY;
            const float top = kv8_group_max(mx);
            const bool moved = top > m[rt] + KVS_LAG;
            if (__any(moved | (rest[rt] > KVS_P_LOG + KVS_V_LAG - vbyte))) {
                const float m_new = moved ? top : m[rt], drop = m[rt] - m_new;
                float most = kv8_group_max(mx - m_new + (float)vbyte);
                most += fabsf(m_new) < KV8_HUGE ? 0.f : fminf(fabsf(m_new) * 0x1p-22f, 64.f);      // the error of m and of a score's product
                const bool over = moved | (most + (float)rest[rt] > 15.f);      // of this row: others' do not change its k
                if (__any(over)) {
                    m[rt] = m_new;
                    l[rt] *= __builtin_amdgcn_exp2f(drop);
                    const float before = (float)rest[rt];
                    rest[rt] = over ? KVS_P_LOG - (int)ceilf(kv8_k(fmaxf(KVS_P_LOG - before + drop, most))) : rest[rt];
                    const float shrink = __builtin_amdgcn_exp2f(drop + ((float)rest[rt] - before));
#pragma unroll
                    for (int i = 0; i < ND; ++i) acc[rt][i] *= shrink;
                }
            }
            const int log = max(rest[rt] + vbyte, (int)KV8_LEAST);
            const float b = (float)log - m[rt];
            float add = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[rt][t][i] = seen > 0 ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][t][i], f, b)) : 0.f;
                    add += s[rt][t][i];
                }
            l[rt] += __builtin_ldexpf(add, -log);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                pr[rt][t >> 1][2 * (t & 1)] = bitcast<uint32_t>(half2_t{(_Float16)s[rt][t][0], (_Float16)s[rt][t][1]});
                pr[rt][t >> 1][2 * (t & 1) + 1] = bitcast<uint32_t>(half2_t{(_Float16)s[rt][t][2], (_Float16)s[rt][t][3]});
            }
        }
        if (!full || __any(v_nan)) {
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                if (16 * i >= D) continue;
                if (v_nan) vr[i] = uint4_t{0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu};      // byte 255: every value of the page
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = min(max(seen - 4 * e, 0), 4);
                    vr[i][e] &= n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            if (16 * i >= D) continue;
            uint4_t op[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) op[u] = kv8_eight<DT_F16>(vr[i][2 * u], vr[i][2 * u + 1], 1.0f);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int u = 0; u < 2; ++u) acc[rt][i] = mx_mfma16<DT_F16>(op[u], pr[rt][u], acc[rt][i]);
        }
        if (more) {
            fetch_v(ci + KVS_WAVES);
            pages(ci + 2 * KVS_WAVES);
        }
    }

    // The waves' parts: maxima, sums and scaled accumulators, [wave][row], in LDS.
    const int pitch = D + 4;
    float *wm = (float *)smem, *wl = wm + KVS_WAVES * ROWS, *wacc = wl + KVS_WAVES * ROWS;      // [wave][ROWS][pitch]
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = kv8_group_sum(l[rt]);
        if (g == 0) {
            wm[wave * ROWS + 16 * rt + col] = m[rt];
            wl[wave * ROWS + 16 * rt + col] = sum;
        }
        float *mine = wacc + (wave * ROWS + 16 * rt + col) * pitch + 4 * g;
        const int unit = -rest[rt] - 127;
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D)
                *(float4_t *)(mine + 16 * i) = float4_t{__builtin_ldexpf(acc[rt][i][0], unit), __builtin_ldexpf(acc[rt][i][1], unit),
                                                        __builtin_ldexpf(acc[rt][i][2], unit), __builtin_ldexpf(acc[rt][i][3], unit)};
    }
    __syncthreads();
    const int rows = min(ROWS, G.rows - w.r0), D4 = D >> 2;
    const int64_t out = (int64_t)w.record * ROWS;
    for (int i = threadIdx.x; i < rows * D4; i += 64 * KVS_WAVES) {
        const int rr = i / D4, d = 4 * (i % D4);
        float tm = wm[rr], tl = 0.f;
#pragma unroll
        for (int k = 1; k < KVS_WAVES; ++k) tm = fmaxf(tm, wm[k * ROWS + rr]);
        float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KVS_WAVES; ++k) {
            const float by = __builtin_amdgcn_exp2f(wm[k * ROWS + rr] - tm);
            tl += wl[k * ROWS + rr] * by;
            v += *(const float4_t *)(wacc + (k * ROWS + rr) * pitch + d) * by;
        }
        *(float4_t *)(a.pre.acc + (out + rr) * D + d) = v;
        if (d == 0) *(float2_t *)(a.pre.ml + (out + rr) * 2) = float2_t{tm, tl};
    }
    __syncthreads();                                 // the waves' parts in LDS have been read
}

template <int QT, int NH, int RT>
__global__ void __launch_bounds__(64 * KVS_WAVES, NH <= 2 && RT == 1 ? 2 : 1)
kv8_prefix_kernel(Kv8Attend a, Kv8Shared x) {
    constexpr int ROWS = 16 * RT;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, H = a.cache.H, heads = H * a.G;
    const uint32_t wgs = gridDim.x, wg = wgs % 8 ? blockIdx.x : blockIdx.x % 8 * (wgs / 8) + blockIdx.x / 8;
    if (x.groups && (x.groups[0] != 0 || x.groups[x.S] != a.batch.B)) {
        // Tokens of no group have no records.
        const int lo = min(max(x.groups[0], 0), a.batch.B), hi = min(max(x.groups[x.S], 0), a.batch.B);
        const int t0 = a.batch.cu ? a.batch.cu[lo] : lo * a.batch.each, t1 = a.batch.cu ? a.batch.cu[hi] : hi * a.batch.each;
        for (int t = wg; t < a.batch.T; t += wgs)
            if (t < t0 || t >= t1)
                for (int i = threadIdx.x; i < heads; i += 64 * KVS_WAVES) a.pre.at[(int64_t)t * heads + i] = int2{0, 0};
    }
    // Pieces, and tiles, of the prefixes 64 at a time; 0xFFFFFFFF: too many (only if tokens are several prefixes').
    auto add = [](uint32_t p, uint32_t q) { return __builtin_elementwise_add_sat(p, q); };
    struct Count { uint32_t pieces, tiles; };
    auto count = [&](int s) -> Count {
        if (s >= x.S) return {0, 0};
        const Kv8Group g = kv8_group<ROWS>(a, x, s);
        return {(uint32_t)g.tiles * (uint32_t)g.pieces, (uint32_t)g.tiles};
    };
    auto scan = [&](uint32_t v) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d);
            if (lane >= d) v = add(v, up);
        }
        return v;
    };
    Count own = count(lane), sum = {scan(own.pieces), scan(own.tiles)};
    uint32_t per_head = __shfl(sum.pieces, 63), tiles = __shfl(sum.tiles, 63);
    for (int s0 = 64; s0 < x.S; s0 += 64) {
        const Count n = count(s0 + lane);
        per_head = add(per_head, __shfl(scan(n.pieces), 63));
        tiles = add(tiles, __shfl(scan(n.tiles), 63));
    }
    if (per_head == 0 || (uint64_t)per_head * (uint32_t)H > 0x7FFFFFFFu || (int64_t)tiles * H + wgs > a.pre.records) return;
    const uint32_t all = per_head * H, least = min((uint32_t)KVS_WAVES, (per_head + x.S - 1) / x.S);
    const uint32_t chunk = max((all + wgs - 1) / wgs, least);
    const uint32_t start = (uint32_t)min((uint64_t)wg * chunk, (uint64_t)all), end = min(start + chunk, all);
    uint32_t before = 0, tiles_before = 0;           // of the 64 prefixes that own and sum are of
    int s0 = 0, head = -1;
    for (uint32_t at = start; at < end;) {
        const int h = (int)(at / per_head);
        const uint32_t in_head = at - h * per_head;
        if (h != head && x.S > 64) {                 // from the first prefix again
            s0 = 0;
            before = tiles_before = 0;
            own = count(lane);
            sum = {scan(own.pieces), scan(own.tiles)};
        }
        head = h;
        uint64_t past;
        while (!(past = __ballot(before + sum.pieces > in_head))) {
            before += __shfl(sum.pieces, 63);
            tiles_before += __shfl(sum.tiles, 63);
            s0 += 64;
            if (s0 >= x.S) return;                   // not reached
            own = count(s0 + lane);
            sum = {scan(own.pieces), scan(own.tiles)};
        }
        const int k = __builtin_ctzll(past);
        const Kv8Group g0 = kv8_group<ROWS>(a, x, s0 + k);
        const Kv8Group g = {kv8_same(g0.first), kv8_same(g0.rows), kv8_same(g0.ctx), kv8_same(g0.tiles), kv8_same(g0.pieces)};
        const uint32_t in_group = kv8_same(in_head - (before + __shfl(sum.pieces, k) - __shfl(own.pieces, k)));
        const uint32_t i = in_group / g.pieces, c0 = in_group - i * g.pieces, n = min((uint32_t)g.pieces - c0, end - at);
        const uint32_t tile = kv8_same(h * tiles + tiles_before + __shfl(sum.tiles, k) - __shfl(own.tiles, k) + i);
        const uint32_t first = at - c0, begun = first / chunk, parts = (first + g.pieces - 1) / chunk - begun + 1;
        const Kv8Part w = {s0 + k, h, (int)i * ROWS, (int)c0, (int)(c0 + n), (int)(tile + wg)};
        if (c0 == 0)
            for (int rr = threadIdx.x; rr < min(ROWS, g.rows - w.r0); rr += 64 * KVS_WAVES) {
                const int r = w.r0 + rr;
                a.pre.at[(int64_t)(g.first + r / a.G) * heads + h * a.G + r % a.G] = int2{(int)(tile + begun) * ROWS + rr, (int)parts};
            }
        kv8_prefix_tile<QT, NH, RT>(a, x, g, w, smem);
        at += n;
    }
}

namespace {
struct Plan { int rt, wgs; int64_t tiles; };
Plan prefix_plan(const Kv8Attend &a, const Kv8Shared &x) {
    Plan p;
    const int64_t rows = (int64_t)a.batch.T * a.G, average = rows / x.S;
    // As many rows at once as the prefixes have, and registers and LDS hold: 64, or 32 where D > 128.
    p.rt = average <= 16 ? 1 : average <= 32 || a.cache.D > 128 ? 2 : 4;
    if (const char *v = opt("MCQ4_KV8_PREFIX_TILES")) p.rt = std::min(a.cache.D > 128 ? 2 : 4, std::max(1, atoi(v)));
    if (p.rt == 3) p.rt = 2;
    p.tiles = (rows / (16 * p.rt) + x.S) * a.cache.H;
    const int64_t seen = std::min<int64_t>((int64_t)x.W << a.cache.page_log, std::max(x.max_prefix, 1)), pieces = (seen + KVD_STEP - 1) / KVD_STEP;
    // As many workgroups as the CUs hold at once.
    p.wgs = (int)std::min<int64_t>(p.rt == 1 && a.cache.D <= 128 ? 512 : 256, p.tiles * pieces);
    if (const char *v = opt("MCQ4_KV8_PREFIX_WGS")) p.wgs = std::max(1, std::min(2048, atoi(v)));
    return p;
}
size_t prefix_lds(int D, int rt) { return KVS_WAVES * 16 * rt * (2 + D + 4) * sizeof(float); }
}  // namespace

size_t kv8_prefix_bytes(const Kv8Attend &a, const Kv8Shared &x, Kv8Prefix *out, void *ws) {
    const Plan p = prefix_plan(a, x);
    const int64_t rows = 16 * p.rt, records = p.tiles + p.wgs, heads = (int64_t)a.cache.H * a.G;
    const size_t acc = (size_t)records * rows * a.cache.D * sizeof(float), ml = (size_t)records * rows * 2 * sizeof(float);
    const size_t at = ((size_t)a.batch.T * heads * sizeof(int2) + 15) / 16 * 16;
    *out = {(int2 *)ws, (float *)((char *)ws + at), (float *)((char *)ws + at + acc), (int)rows, records};
    return at + acc + ml;
}

template <int QT, int NH, int RT>
static hipError_t launch_kv8_prefix_t(const Kv8Attend &a, const Kv8Shared &x, const Plan &p, hipStream_t s) {
    const size_t lds = prefix_lds(a.cache.D, RT);
    static std::atomic<uint64_t> done{0};
    if (lds > 64 * 1024)
        if (hipError_t e = mx_allow_lds((const void *)kv8_prefix_kernel<QT, NH, RT>, 160 * 1024, done)) return e;
    hipLaunchKernelGGL((kv8_prefix_kernel<QT, NH, RT>), dim3((unsigned)p.wgs), dim3(64 * KVS_WAVES), lds, s, a, x);
    return hipGetLastError();
}
template <int QT, int NH>
static hipError_t launch_kv8_prefix_n(const Kv8Attend &a, const Kv8Shared &x, const Plan &p, hipStream_t s) {
    if (p.rt == 1) return launch_kv8_prefix_t<QT, NH, 1>(a, x, p, s);
    if constexpr (NH <= 2)
        if (p.rt == 4) return launch_kv8_prefix_t<QT, NH, 4>(a, x, p, s);
    return launch_kv8_prefix_t<QT, NH, 2>(a, x, p, s);
}
template <int QT>
static hipError_t launch_kv8_prefix_q(const Kv8Attend &a, const Kv8Shared &x, const Plan &p, hipStream_t s) {
    switch ((a.cache.D + 63) / 64) {
        case 1: return launch_kv8_prefix_n<QT, 1>(a, x, p, s);
        case 2: return launch_kv8_prefix_n<QT, 2>(a, x, p, s);
        case 3: return launch_kv8_prefix_n<QT, 3>(a, x, p, s);
        default: return launch_kv8_prefix_n<QT, 4>(a, x, p, s);
    }
}
hipError_t launch_kv8_prefix(const Kv8Attend &a, const Kv8Shared &x, hipStream_t s) {
    const Plan p = prefix_plan(a, x);
    return a.q_dt == DT_BF16 ? launch_kv8_prefix_q<DT_BF16>(a, x, p, s) : launch_kv8_prefix_q<DT_F16>(a, x, p, s);
}

}  // namespace mcq4
