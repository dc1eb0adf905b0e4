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
// fp32.  V's is applied by the conversion, relative to the largest one the wave has met, which
// multiplies the accumulators in the end: fp16 then holds every code of pages within 2^8 of the
// largest scale exactly, and P in fp16 (11 bits) is the only operand that is rounded.
//
// A masked score is -inf whatever K holds there, but 0 times a NaN of V would be NaN: tiles with
// a masked token look for NaN codes, zero them, and set the rows that do attend to one to NaN.
//
// The context is dealt out over workgroups (a span of whole 64-token pieces each) and in them
// over four waves; kv8_join_kernel adds the workgroups' parts up in order.
#include <algorithm>

#include "kv8_common.h"

namespace mcq4 {

constexpr int KVD_WAVES = 4, KVD_ROWS = 16, KVD_STEP = 64;
constexpr float LOG2E = 1.4426950408889634f;

struct Kv8Plan {
    int tiles_each;      // row tiles per sequence, or 0: offsets given, looked up
    int tiles;           // upper bound over all sequences
    int splits, span;    // parts of a context, and the 64-token pieces of one
    float *acc;          // [tiles][H][splits][16][D]
    float *ml;           // [tiles][H][splits][16][2]
};

template <int QT>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w, float s, bool high) {
    if constexpr (QT == DT_BF16) {
        return high ? bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))
                    : bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
    } else {
        return high ? bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true))
                    : bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false));
    }
}
// Eight codes (two dwords) as an MFMA operand.
template <int QT>
__device__ __forceinline__ uint4_t kv8_eight(uint32_t lo, uint32_t hi, float s) {
    uint4_t r = {kv8_pair<QT>(lo, s, false), kv8_pair<QT>(lo, s, true), kv8_pair<QT>(hi, s, false), kv8_pair<QT>(hi, s, true)};
    return r;
}
// 0xFF in every byte whose code is NaN (0x7F, 0xFF).
__device__ __forceinline__ uint32_t kv8_nan_bytes(uint32_t w) {
    const uint32_t t = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    return (t >> 7) * 0xFFu;
}
__device__ __forceinline__ float kv8_group_max(float x) {      // over the four lanes l % 16 + 16 g
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float kv8_group_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// What a tile of rows covers of its sequence.
struct Kv8Rows {
    int b, r0, rows;      // sequence, first row, rows of the sequence
    int first_token;      // of the sequence's new tokens
    int ctx, pos0;        // context, position of new token 0
    int lo, hi;           // pieces of 64 tokens that any row of the tile sees: [lo, hi)
};

__device__ __forceinline__ bool kv8_rows(const Kv8Attend &a, const Kv8Plan &p, int tile, int tile_rows, Kv8Rows &o) {
    Kv8Item it;
    if (p.tiles_each) it = {tile / p.tiles_each, tile % p.tiles_each};
    else it = kv8_locate(tile, a.batch.B, [&](int b) { return (kv8_span(a.batch, b).n * a.G + tile_rows - 1) / tile_rows; });
    if (it.b >= a.batch.B) return false;
    const Kv8Span sp = kv8_span(a.batch, it.b);
    o.b = it.b;
    o.r0 = it.i * tile_rows;
    o.rows = sp.n * a.G;
    o.first_token = sp.first;
    if (o.r0 >= o.rows) return false;
    const int most = a.batch.W << a.cache.page_log;
    o.ctx = min(max(a.batch.lens[it.b], 0), most);
    // A context that holds fewer tokens than are new: the first of them stand before it and see nothing.
    o.pos0 = o.ctx - sp.n;
    const int last = (min(o.r0 + tile_rows, o.rows) - 1) / a.G;
    const int end = a.causal ? min(max(o.pos0 + last + 1, 0), o.ctx) : o.ctx;
    const int begin = a.window ? max(o.pos0 + o.r0 / a.G - a.window + 1, 0) : 0;
    o.lo = begin / KVD_STEP;
    o.hi = end > begin ? (end + KVD_STEP - 1) / KVD_STEP : o.lo;
    return true;
}

template <int QT, int NH>
__global__ void __launch_bounds__(64 * KVD_WAVES)
kv8_attend_kernel(Kv8Attend a, Kv8Plan p) {
    constexpr int ND = 4 * NH;                      // channel tiles of 16
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits, h = blockIdx.y;
    Kv8Rows R;
    if (!kv8_rows(a, p, tile, KVD_ROWS, R)) return;
    const int pieces = R.hi - R.lo;
    const int parts = max(1, min(p.splits, (pieces + p.span - 1) / p.span));
    if (split >= parts) return;
    const int c0 = R.lo + split * p.span, c1 = split == parts - 1 ? R.hi : c0 + p.span;

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
    int vref = 0;                                   // scale byte that the accumulators are relative to
    const float qk = a.scale * LOG2E;

    const int k_sub = 16 * (col >> 2) + (col & 3);  // K row of tile a: token k_sub + 4 a
    uint4_t kr[4][NH], vr[ND];
    int vbyte = 0;
    float kscale = 0.f;
    // The scales, K and V of piece ci.  Groups without tokens read page 0, whose bytes are not used.
    auto fetch = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        const int tk = t0 + 16 * (col >> 2), tv = t0 + 16 * g;
        int pk = tk < R.ctx ? kv8_page(a.batch, c.P, page_log, R.b, tk) : -1;
        int pv = tv < R.ctx ? kv8_page(a.batch, c.P, page_log, R.b, tv) : -1;
        const bool ok = pv >= 0;
        pk = max(pk, 0);
        pv = max(pv, 0);
        const int64_t bk = (int64_t)pk * c.H + h, bv = (int64_t)pv * c.H + h;
        const uint32_t kb = c.ks[bv], vb = c.vs[bv];
        const uint8_t *kp = c.k + bk * page * D + (int64_t)((t0 + k_sub) & (page - 1)) * D + 16 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < NH; ++i)
                kr[t][i] = 64 * i + 16 * g < D ? *(const uint4_t *)(kp + 4 * t * D + 64 * i) : uint4_t{0, 0, 0, 0};
        const uint8_t *vp = c.v + bv * page * D + (int64_t)col * page + (tv & (page - 1));
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D) vr[i] = *(const uint4_t *)(vp + (int64_t)16 * i * page);
        // A page that is not there: nothing of it is seen (kscale < 0 marks it).
        kscale = ok ? qk * __uint_as_float(kb << 23) : NAN;
        vbyte = ok ? (int)vb : 0;
        return ok;
    };

    for (int ci = c0 + wave; ci < c1; ci += KVD_WAVES) {
        const bool here = fetch(ci);
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
        const float m_new = fmaxf(m, kv8_group_max(mx)), m_use = m_new == -INFINITY ? 0.f : m_new;
        float shrink = __builtin_amdgcn_exp2f(m - m_use);
        m = m_new;
        l *= shrink;
        if (__any(vbyte > vref)) {
            int top = max(vbyte, __shfl_xor(vbyte, 16));
            top = max(max(top, __shfl_xor(top, 32)), vref);
            const int e = vref - top;
            shrink *= e < -126 ? 0.f : __uint_as_float((uint32_t)(e + 127) << 23);
            vref = top;
        }
        float add = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - m_use);
                add += s[t][i];
            }
        l += add;
        uint4_t pv[2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            pv[t >> 1][2 * (t & 1)] = bitcast<uint32_t>(half2_t{(_Float16)s[t][0], (_Float16)s[t][1]});
            pv[t >> 1][2 * (t & 1) + 1] = bitcast<uint32_t>(half2_t{(_Float16)s[t][2], (_Float16)s[t][3]});
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] *= shrink;
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
        // Below vref the factor is a power of two of at most 1; far below it is 0 and so are the values.
        const int rel = vbyte - vref;
        const float vs = rel < -100 ? 0x1p-100f : __uint_as_float((uint32_t)(rel + 127) << 23);
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (16 * i < D)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    acc[i] = mx_mfma16<DT_F16>(kv8_eight<DT_F16>(vr[i][2 * u], vr[i][2 * u + 1], vs), pv[u], acc[i]);
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
    // exp2 of a maximum that is NaN stays NaN through the sums.
    float f = __builtin_amdgcn_exp2f(m - t_use);
    if (vref > 0) f *= __uint_as_float((uint32_t)vref << 23);
    float *mine = wacc + (wave * 16 + col) * pitch + 4 * g;
#pragma unroll
    for (int i = 0; i < ND; ++i)
        if (16 * i < D) *(float4_t *)(mine + 16 * i) = acc[i] * f;
    __syncthreads();
    const int rows = min(KVD_ROWS, R.rows - R.r0), D4 = D >> 2;
    const int64_t part = ((int64_t)tile * c.H + h) * p.splits + split;
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
        if (parts > 1) {
            *(float4_t *)(p.acc + (part * 16 + rr) * D + d) = v;
            if (d == 0) {
                p.ml[(part * 16 + rr) * 2] = tm;
                p.ml[(part * 16 + rr) * 2 + 1] = tl;
            }
            continue;
        }
        const int rt = (R.r0 + rr) / a.G, rh = h * a.G + (R.r0 + rr) % a.G;
        const int64_t o = ((int64_t)(R.first_token + rt) * c.H * a.G + rh);
        const float inv = tl == 0.f ? 0.f : 1.0f / tl;      // a row that sees nothing is 0
#pragma unroll
        for (int e = 0; e < 4; ++e) mx_store<QT>(a.out, o * D + d + e, v[e] * inv);
        if (a.lse && d == 0) a.lse[o] = tl == 0.f ? -INFINITY : (tm + __builtin_amdgcn_logf(tl)) * (1.0f / LOG2E);
    }
}

// One wave per row: the parts of its context, in order.
template <int QT>
__global__ void __launch_bounds__(256)
kv8_join_kernel(Kv8Attend a, Kv8Plan p) {
    const Kv8Cache &c = a.cache;
    const int lane = threadIdx.x & 63, h = blockIdx.y;
    const int tile = blockIdx.x >> 2, rr = 4 * (blockIdx.x & 3) + (threadIdx.x >> 6);
    Kv8Rows R;
    if (!kv8_rows(a, p, tile, KVD_ROWS, R) || R.r0 + rr >= R.rows) return;
    const int parts = min(p.splits, (R.hi - R.lo + p.span - 1) / p.span);
    if (parts <= 1) return;                        // written by its only part
    const int64_t base = ((int64_t)tile * c.H + h) * p.splits;
    float top = -INFINITY;
    for (int s = lane; s < parts; s += 64) top = fmaxf(top, p.ml[((base + s) * 16 + rr) * 2]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float use = top == -INFINITY ? 0.f : top;
    float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) {
        const int64_t at = (base + s) * 16 + rr;
        const float w = __builtin_amdgcn_exp2f(p.ml[at * 2] - use);
        l += p.ml[at * 2 + 1] * w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < c.D) v[i] += p.acc[at * c.D + lane + 64 * i] * w;
    }
    const int rt = (R.r0 + rr) / a.G, rh = h * a.G + (R.r0 + rr) % a.G;
    const int64_t o = (int64_t)(R.first_token + rt) * c.H * a.G + rh;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < c.D) mx_store<QT>(a.out, o * c.D + lane + 64 * i, v[i] * inv);
    if (a.lse && lane == 0) a.lse[o] = l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * (1.0f / LOG2E);
}

static Kv8Plan kv8_plan(const Kv8Attend &a) {
    Kv8Plan p;
    const Kv8Batch &b = a.batch;
    p.tiles_each = b.cu ? 0 : (b.each * a.G + KVD_ROWS - 1) / KVD_ROWS;
    p.tiles = b.cu ? (int)(((int64_t)b.T * a.G) / KVD_ROWS + b.B) : b.B * p.tiles_each;
    int64_t seen = std::min<int64_t>((int64_t)b.W << a.cache.page_log, a.max_context);
    if (a.window && !b.cu) seen = std::min<int64_t>(seen, (int64_t)a.window + b.each + 2 * KVD_STEP);
    const int64_t pieces = std::max<int64_t>(1, (seen + KVD_STEP - 1) / KVD_STEP);
    const int64_t wgs = (int64_t)p.tiles * a.cache.H;
    // About 1024 workgroups, of at least two pieces for each wave.
    int64_t splits = std::min<int64_t>((1024 + wgs - 1) / wgs, (pieces + 2 * KVD_WAVES - 1) / (2 * KVD_WAVES));
    splits = std::max<int64_t>(1, std::min<int64_t>(splits, 256));
    p.span = (int)((pieces + splits - 1) / splits);
    p.splits = (int)((pieces + p.span - 1) / p.span);
    p.acc = p.ml = nullptr;
    return p;
}

size_t kv8_attend_workspace_bytes(const Kv8Attend &a) {
    const Kv8Plan p = kv8_plan(a);
    if (p.splits == 1) return 0;
    return (size_t)p.tiles * a.cache.H * p.splits * 16 * (a.cache.D + 2) * sizeof(float);
}

template <int QT, int NH>
static hipError_t launch_kv8_attend_t(const Kv8Attend &a, Kv8Plan p, hipStream_t s) {
    const size_t lds = KVD_WAVES * 16 * (2 + a.cache.D + 4) * sizeof(float);
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void *)kv8_attend_kernel<QT, NH>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((kv8_attend_kernel<QT, NH>), dim3((unsigned)p.tiles * p.splits, (unsigned)a.cache.H), dim3(64 * KVD_WAVES), lds, s, a, p);
    if (p.splits > 1)
        hipLaunchKernelGGL(kv8_join_kernel<QT>, dim3((unsigned)p.tiles * 4, (unsigned)a.cache.H), dim3(256), 0, s, a, p);
    return hipGetLastError();
}

template <int QT>
static hipError_t launch_kv8_attend_q(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s) {
    switch ((a.cache.D + 63) / 64) {
        case 1: return launch_kv8_attend_t<QT, 1>(a, p, s);
        case 2: return launch_kv8_attend_t<QT, 2>(a, p, s);
        case 3: return launch_kv8_attend_t<QT, 3>(a, p, s);
        default: return launch_kv8_attend_t<QT, 4>(a, p, s);
    }
}

hipError_t launch_kv8_attend(const Kv8Attend &a, void *ws, hipStream_t s) {
    Kv8Plan p = kv8_plan(a);
    if (p.splits > 1) {
        p.acc = (float *)ws;
        p.ml = p.acc + (size_t)p.tiles * a.cache.H * p.splits * 16 * a.cache.D;
    }
    return a.q_dt == DT_BF16 ? launch_kv8_attend_q<DT_BF16>(a, p, s) : launch_kv8_attend_q<DT_F16>(a, p, s);
}

}  // namespace mcq4
