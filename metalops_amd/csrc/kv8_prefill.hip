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
#include <type_traits>

#include "kv8_attend.h"

namespace mcq4 {

constexpr int KVP_WAVE_ROWS = 32;
// P's largest is at 2^KVP_P_LOG where m and k have just followed, and at most 2^15 else: scores may exceed m by KVP_LAG and
// a page's scale k by KVP_V_LAG, beyond which a half's parts of the output are looked at themselves.  2048 of 4096 and 1500
// of 1500 tokens, 32 heads, D = 128, keys with channels eight times larger: 154.7 us with 7 and 1, 156.0 with 6 and 1,
// 158.7 with 5 and 1; with even keys 5 to 7 make no difference, 2 costs 7% and no lag of the scale 2%.
constexpr int KVP_LAG = 7, KVP_V_LAG = 1, KVP_P_LOG = 15 - KVP_LAG - KVP_V_LAG;
constexpr int KVP_V_PITCH = KVD_STEP * 2 + 16;
constexpr int kvp_ahead(int NT) { return NT % 2 == 0 ? (NT == 2 ? 2 : 4) : NT == 3 ? 3 : 2; }     // a divisor of 2 NT
constexpr int kvp_waves(int NT) { return NT <= 4 ? 8 : 4; }
constexpr int kvp_channels(int NT) { return NT <= 4 ? 128 : NT <= 6 ? 192 : 256; }     // in LDS: every thread's part
constexpr int kvp_k_buffers(int NT) { return NT <= 6 ? 3 : 2; }      // D > 192: LDS holds no more
constexpr int kvp_k_pitch(int NT) { return 2 * kvp_channels(NT) + 16; }
constexpr int kvp_k_bytes(int NT) { return KVD_STEP * kvp_k_pitch(NT); }
constexpr int kvp_v_bytes(int NT) { return kvp_channels(NT) * KVP_V_PITCH; }

__device__ __forceinline__ float kvp_other(float x) {      // the value of lane l ^ 32
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? p[0] : p[1]);
}

template <int QT>
__device__ __forceinline__ float16_t kvp_mfma(uint4_t a, uint4_t b, float16_t c) { return mfma32<QT>(bitcast<half8_t>(a), bitcast<half8_t>(b), c); }

// 16 codes as 16-bit values, to 32 bytes of LDS.
template <int QT>
__device__ __forceinline__ void kvp_put(uint8_t *dst, uint4_t w) {
    *(uint4_t *)dst = kv8_eight<QT>(w[0], w[1], 1.0f);
    *(uint4_t *)(dst + 16) = kv8_eight<QT>(w[2], w[3], 1.0f);
}

// The error of m, of log - m and of a score's product, where their steps are 1 or more.
__device__ __forceinline__ float kvp_room(float m) { return fabsf(m) < KV8_HUGE ? 0.f : fminf(fabsf(m) * 0x1p-22f, 64.f); }

// NT: tiles of 32 channels.
template <int QT, int NT>
__global__ void __launch_bounds__(64 * kvp_waves(NT), 1)
kv8_prefill_kernel(Kv8Attend a, Kv8Plan p) {
    constexpr int WAVES = kvp_waves(NT), ROWS = KVP_WAVE_ROWS * WAVES, CH = kvp_channels(NT);
    constexpr int KL = WAVES, NC = CH / (16 * KL);       // threads of a K token; 16-byte pieces of K, and of V, of a thread
    constexpr int KB = kvp_k_buffers(NT), K_PITCH = kvp_k_pitch(NT), K_BYTES = kvp_k_bytes(NT), V_BYTES = kvp_v_bytes(NT);
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ int nan_flag[2];
    __shared__ __attribute__((aligned(8))) uint16_t nan_map[2][CH][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hi = lane >> 5;
    // Neighbouring workgroups take neighbouring heads: with 8 of them an XCD's L2 serves one.
    const int h = (int)(blockIdx.x % (uint32_t)a.cache.H), tile = (int)(blockIdx.x / (uint32_t)a.cache.H);
    if (a.batch.cu && blockIdx.y == 0) kv8_rest(a, blockIdx.x, gridDim.x);
    Kv8Rows R;
    if (!kv8_longest_first(a, tile, ROWS, R)) return;
    kv8_uniform(R);
    const int split = blockIdx.y, parts = kv8_parts(R, p);
    if (split >= parts) return;
    const int c0 = R.lo + split * p.span, c1 = split == parts - 1 ? R.hi : c0 + p.span;

    const Kv8Cache &c = a.cache;
    const int D = c.D, page_log = c.page_log, page = 1 << page_log;
    // This lane's row, and what it and the wave's see.
    const int w0 = min(R.r0 + KVP_WAVE_ROWS * wave, R.rows - 1), w1 = min(R.r0 + KVP_WAVE_ROWS * (wave + 1), R.rows) - 1;
    const bool rows_here = R.r0 + KVP_WAVE_ROWS * wave < R.rows;
    const int r = min(R.r0 + KVP_WAVE_ROWS * wave + col, R.rows - 1), tok = r / a.G, pos = R.pos0 + tok;
    const int see_hi = a.causal ? min(pos + 1, R.ctx) : R.ctx;
    const int see_lo = a.window ? max(pos - a.window + 1, 0) : 0;
    const int pos_a = R.pos0 + w0 / a.G, pos_z = R.pos0 + max(w1, w0) / a.G;
    const int all_hi = a.causal ? pos_a + 1 : R.ctx, all_lo = a.window ? pos_z - a.window + 1 : 0;
    const int any_hi = a.causal ? min(pos_z + 1, R.ctx) : R.ctx, any_lo = a.window ? pos_a - a.window + 1 : 0;
    // What all rows of the workgroup see (a page that is missing aside).
    const int tile_hi = a.causal ? min(R.pos0 + R.r0 / a.G + 1, R.ctx) : R.ctx;
    const int tile_lo = a.window ? R.pos0 + (min(R.r0 + ROWS, R.rows) - 1) / a.G - a.window + 1 : 0;
    auto seen_by_wave = [&](int ci) { return rows_here && ci < c1 && ci * KVD_STEP < any_hi && (ci + 1) * KVD_STEP > any_lo; };

    // A negative scale goes into q's sign: the scores' factor is positive, and a maximum stays one.
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    uint4_t qv[2 * NT];
    const uint16_t *q = (const uint16_t *)a.q + (int64_t)(R.first_token + tok) * a.q_token + (int64_t)(h * a.G + r % a.G) * a.q_head;
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
    float m = -__FLT_MAX__, l = 0.f;                     // m is finite from the start: no score, masked ones included, needs a case of its own
    int rest = KVP_P_LOG - (int)KV8_NO_K;                // KVP_P_LOG - k; a new k comes from the last one, relative to the new m
    const float qk = fabsf(a.scale) * LOG2E;

    // The thread's part of a piece: K token tid / KL (a wave's lie in one page), 16-byte pieces
    // tid % KL + KL i; V channels tid / 4 + 16 WAVES i, tokens 16 (tid % 4) ..  Channels past D
    // repeat the last ones: q is 0 there, and those of V are not stored.  Scale bytes are those
    // of tokens 16 (tid % 4) ..: K's in bits 0..7 of kb, V's in 16..23, bit 8 for a page that is not there.
    uint4_t kr[NC], vr[NC];
    // Table entries: ek, es of the next K to be fetched (its codes, its scales), ev of the next V.
    // Nothing branches on them, and they are loaded in every iteration, so that no load is waited
    // for before the next one.
    int ek, es, ev;
    uint32_t kb_next = 0, vb_next = 0, kb_now = 0;
    bool k_there = false, v_there = false;
    const uint8_t *const table = (const uint8_t *)(a.batch.table + R.b * a.batch.table_stride);
    const uint32_t pages = (uint32_t)c.P, page_codes = (uint32_t)(c.H * page * D);      // fit 31 bits (checked at the C entry)
    const int quarter = tid & 3, k_line = (int)((uint32_t)tid / KL), k_part = (int)((uint32_t)tid % KL), line = tid >> 2;
    // A piece begins at a page or inside one, and page sizes are powers of two: the parts of a token's place add up.
    const uint32_t k_entry = k_line >> page_log, s_entry = (16 * quarter) >> page_log, last_entry = a.batch.W - 1;
    auto entries = [&](int ci) {
        const uint32_t first = (uint32_t)(ci * KVD_STEP) >> page_log;
        ev = es;
        ek = *(const int *)(table + 4 * min(first + k_entry, last_entry));
        es = *(const int *)(table + 4 * min(first + s_entry, last_entry));
    };
    const int ctx_part = R.ctx - 16 * quarter;
    const uint8_t *const k_at = c.k + (uint32_t)h * page * D + (k_line & (page - 1)) * D;
    const uint8_t *const v_at = c.v + (uint32_t)h * page * D + ((16 * quarter) & (page - 1));
    const uint8_t *const ks_at = c.ks + h, *const vs_at = c.vs + h;
    auto fetch_k = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        const uint32_t idk = (uint32_t)ek < pages ? (uint32_t)ek : 0u;       // codes of a page that is not there: not seen
        k_there = ((uint32_t)es < pages) & (t0 < ctx_part);
        const uint64_t scale = (uint64_t)(k_there ? (uint32_t)es : 0u) * (uint32_t)c.H;
        kb_next = ks_at[scale];
        vb_next = vs_at[scale];
        const uint8_t *kp = k_at + (uint64_t)idk * page_codes + (uint32_t)((t0 & (page - 1)) * D);
#pragma unroll
        for (int i = 0; i < NC; ++i) kr[i] = *(const uint4_t *)(kp + (uint32_t)min(16 * (k_part + KL * i), D - 16));
    };
    auto fetch_v = [&](int ci) {
        const int t0 = ci * KVD_STEP;
        v_there = ((uint32_t)ev < pages) & (t0 < ctx_part);
        const uint32_t id = v_there ? (uint32_t)ev : 0u;
        const uint8_t *vp = v_at + (uint64_t)id * page_codes + (uint32_t)(t0 & (page - 1));
#pragma unroll
        for (int i = 0; i < NC; ++i) vr[i] = *(const uint4_t *)(vp + (uint32_t)(min(line + 16 * WAVES * i, D - 1) << page_log));
    };
    auto put_k = [&](int buf, int i) {
        kvp_put<QT>(smem + buf * K_BYTES + k_line * K_PITCH + 32 * k_part + 32 * KL * i, kr[i]);
    };
    uint32_t largest = 0;                                // byte met; 255, NaN, is for the end
    auto bytes = [&]() {
        largest = max(largest, max(kb_next, vb_next));
        return k_there ? kb_next | vb_next << 16 : 256u;
    };
    // V: first (i = 0) what concerns all of the thread's pieces.
    auto put_v = [&](int buf, int piece, int i) {
        if (i == 0) {
            if (!__all(v_there)) {                           // what page 0 holds there is not seen
#pragma unroll
                for (int k = 0; k < NC; ++k)
                    if (!v_there) vr[k] = uint4_t{0, 0, 0, 0};
            }
            if (piece * KVD_STEP < tile_lo || (piece + 1) * KVD_STEP > tile_hi) {
                // Not every row sees every token: NaN of V would reach rows by 0 * NaN.  They become 0, and a map of
                // them, 64 tokens a channel, says which rows get one (NaN codes elsewhere are NaN by themselves).
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    uint32_t map = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t bad = ((vr[k][e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                        vr[k][e] &= ~((bad >> 7) * 0xFFu);
                        map |= (((bad >> 7) * 0x10204080u) >> 28) << (4 * e);
                    }
                    nan_map[buf][line + 16 * WAVES * k][quarter] = (uint16_t)map;
                    if (map) nan_flag[buf] = piece + 1;
                }
            }
        }
        kvp_put<DT_F16>(smem + KB * K_BYTES + buf * V_BYTES + (line + 16 * WAVES * i) * KVP_V_PITCH + 32 * quarter, vr[i]);
    };

    // K row of S-tile row l % 32: rows 16 j + 8 e + 4 h + i are tokens 16 j + 8 h + 4 e + i.
    const int k_row = (col & 16) | ((col & 4) << 1) | ((col & 8) >> 1) | (col & 3);
    const uint32_t lds0 = lds_addr(smem);
    const uint32_t k_off = lds0 + k_row * K_PITCH + 16 * hi, v_off = lds0 + KB * K_BYTES + col * KVP_V_PITCH + 16 * hi;
    auto read_k = [&](int buf, int t, int k) { return mx_lds16(k_off + buf * K_BYTES + 32 * t * K_PITCH + 32 * k); };
    auto read_v = [&](int buf, int g, int i) { return mx_lds16(v_off + buf * V_BYTES + 32 * i * KVP_V_PITCH + 32 * g); };

    // Raw scores of 32 tokens (sa: a piece's first half, sb: its second); by 16 of them the factor
    // that makes them logarithms to base 2 (never 0: masked ones are -inf) and the scale byte of V;
    // which of them a row sees (bit e: register e); their maximum.
    float16_t sa, sb, zero;
#pragma unroll
    for (int e = 0; e < 16; ++e) zero[e] = 0.f;
    struct Half {
        float f[2], mx;
        int v[2];
        uint32_t seen;
    };
    Half ha, hb;
    // Operands of K and V, read AHEAD products before their use: those of a half's S, of its product with V, and so on.
    constexpr int N = 2 * NT, AHEAD = kvp_ahead(NT), NW = 8;
    static_assert(N % AHEAD == 0, "operands keep their places");
    uint4_t op[AHEAD];
    auto first_operands = [&](int buf) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) op[i] = read_k(buf, 1, i);
    };
    // Of the scores x of half t of piece ci, whose scale bytes are kb: the factors, and the masked ones to -inf.
    auto mask = [&](int ci, int t, uint32_t kb, float16_t &x, Half &o) {
        const int t0 = ci * KVD_STEP + 32 * t;
        const uint32_t k0 = (uint32_t)__builtin_amdgcn_readlane((int)kb, 2 * t), k1 = (uint32_t)__builtin_amdgcn_readlane((int)kb, 2 * t + 1);
        o.f[0] = fmaxf(qk * __uint_as_float((k0 & 255u) << 23), 0x1p-126f);
        o.f[1] = fmaxf(qk * __uint_as_float((k1 & 255u) << 23), 0x1p-126f);
        // Of a page that is not there, whose scores are all masked: as its neighbour's.
        o.v[0] = ((k0 & 256u ? k1 : k0) >> 16) & 255;
        o.v[1] = ((k1 & 256u ? k0 : k1) >> 16) & 255;
        o.seen = 0xFFFFu;
        if (t0 < all_lo || t0 + 32 > all_hi || ((k0 | k1) & 256u)) {
            uint32_t some = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int at = t0 + 16 * j + 8 * hi, from = min(max(see_lo - at, 0), 8), to = min(max(see_hi - at, 0), 8);
                some |= ((j ? k1 : k0) & 256u ? 0u : ((1u << to) - 1) & ~((1u << from) - 1)) << (8 * j);
            }
            o.seen = some;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t keep = (uint32_t)((int)(some << (31 - e)) >> 31);
                x[e] = __uint_as_float((__float_as_uint(x[e]) & keep) | (0xFF800000u & ~keep));
            }
        }
    };
    auto group_max = [&](const float16_t &x, int j) {
        float v = x[8 * j];
#pragma unroll
        for (int e = 1; e < 8; ++e) v = fmaxf(v, x[8 * j + e]);
        return v;
    };
    // All of that for a half whose S nothing runs beside.
    auto scores = [&](int ci, int buf, uint32_t kb, float16_t &x, Half &o) {
#pragma unroll
        for (int k = 0; k < 2 * NT; ++k)
            x = kvp_mfma<QT>(read_k(buf, 0, k), qv[k], k == 0 ? zero : x);
        mask(ci, 0, kb, x, o);
        o.mx = fmaxf(group_max(x, 0) * o.f[0], group_max(x, 1) * o.f[1]);
        o.mx = fmaxf(o.mx, kvp_other(o.mx));
    };

    uint32_t kb_piece = 0;                               // scale bytes of the piece; kb_now: of the next one
    if (tid < 2) nan_flag[tid] = 0;                      // piece + 1 where a buffer's V has a NaN
    if (c0 < c1) {
        es = 0;
        entries(c0);
        fetch_k(c0);
        entries(c0 + 1);
#pragma unroll
        for (int i = 0; i < NC; ++i) put_k(0, i);
        kb_piece = bytes();
        fetch_k(c0 + 1);
        fetch_v(c0);
        entries(c0 + 2);
        __syncthreads();
        if (seen_by_wave(c0)) scores(c0, 0, kb_piece, sa, ha);
        first_operands(0);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            put_k(1, i);
            put_v(0, c0, i);
        }
        kb_now = bytes();
    }
    wait_vmcnt<0>();                                     // q too: nothing in the loop waits for it again
    // The piece's K in buffer b0, the next one's in b1; the one after goes to b2, last read (as the piece's) before
    // this piece's barrier.  With two buffers that is b0, and another barrier stands between the halves.
    int b0 = 0, b1 = 1, b2 = KB == 3 ? 2 : 0;
    for (int ci = c0; ci < c1; ++ci) {
        const int buf = (ci - c0) & 1;
        const bool more = ci + 1 < c1;
        fetch_k(ci + 2);                                 // at the end: of pieces that are not used
        fetch_v(ci + 1);
        entries(ci + 3);
        lds_barrier();                                   // V of the piece and K of the next are there, the other buffers have been read
        const bool has_nan = nan_flag[buf] == ci + 1;
        if (seen_by_wave(ci)) {
            // T = 0: the weights of x = sa, S and maxima of y = sb.  T = 1: the weights of sb, S and maxima of the next
            // piece's sa, and the piece after's K and the next one's V to LDS.
            auto half = [&](auto tt, float16_t &x, Half &hx, float16_t &y, Half &hy) {
                constexpr int T = decltype(tt)::value;
                const bool moved = hx.mx > m + KVP_LAG;
                if (__any(moved | (rest > KVP_P_LOG + KVP_V_LAG - max(hx.v[0], hx.v[1])))) {
                    const float m_new = moved ? hx.mx : m, drop = m - m_new;
                    float most = hx.mx - m_new + (float)hx.v[0];
                    if (hx.v[0] != hx.v[1]) {
                        most = fmaxf(group_max(x, 0) * hx.f[0] - m_new + (float)hx.v[0], group_max(x, 1) * hx.f[1] - m_new + (float)hx.v[1]);
                        most = fmaxf(most, kvp_other(most));
                    }
                    most += kvp_room(m_new);
                    const bool over = moved | (most + (float)rest > 15.f);      // of this row: others' do not change its k
                    if (__any(over)) {
                        m = m_new;
                        l *= __builtin_amdgcn_exp2f(drop);
                        const float before = (float)rest;
                        rest = over ? KVP_P_LOG - (int)ceilf(kv8_k(fmaxf(KVP_P_LOG - before + drop, most))) : rest;
                        const float shrink = __builtin_amdgcn_exp2f(drop + ((float)rest - before));
#pragma unroll
                        for (int i = 0; i < NT; ++i) acc[i] *= shrink;
                    }
                }
                int log[2];
                float b[2], add[2] = {0.f, 0.f};
                log[0] = log[1] = max(rest + hx.v[0], (int)KV8_LEAST);
                b[0] = b[1] = (float)log[0] - m;
                if (hx.v[0] != hx.v[1]) {
                    log[1] = max(rest + hx.v[1], (int)KV8_LEAST);
                    b[1] = (float)log[1] - m;
                }
                const int kbuf = T ? b1 : b0;
                uint4_t pr[2];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    y = kvp_mfma<QT>(op[i % AHEAD], qv[i], i == 0 ? zero : y);
                    if (i + AHEAD < N) op[i % AHEAD] = read_k(kbuf, 1 - T, i + AHEAD);
                    else op[i % AHEAD] = read_v(buf, 2 * T + (i + AHEAD - N) / NT, (i + AHEAD - N) % NT);
#pragma unroll
                    for (int w = 0; w < NW; ++w)
                        if (w * N / NW == i) {
                            const int j = w >> 2, e = 2 * w;
                            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], hx.f[j], b[j]));
                            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e + 1], hx.f[j], b[j]));
                            add[j] += p0 + p1;
                            // opaque: else the compiler moves the exponentials to where P is used
                            pr[j][w & 3] = opaque_vgpr(bitcast<uint32_t>(half2_t{(_Float16)p0, (_Float16)p1}));
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (hx.v[0] == hx.v[1]) l += __builtin_ldexpf(add[0] + add[1], -log[0]);
                else l += __builtin_ldexpf(add[0], -log[0]) + __builtin_ldexpf(add[1], -log[1]);
                const bool next = T == 0 || more;
                if (next) mask(T ? ci + 1 : ci, 1 - T, T ? kb_now : kb_piece, y, hy);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    acc[i % NT] = kvp_mfma<DT_F16>(op[i % AHEAD], pr[i / NT], acc[i % NT]);
                    if (i + AHEAD < N) op[i % AHEAD] = read_v(buf, 2 * T + (i + AHEAD) / NT, (i + AHEAD) % NT);
                    else op[i % AHEAD] = read_k(b1, T, i + AHEAD - N);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (N / 4 + k * N / 4 == i) {
                            const float v = group_max(y, k) * hy.f[k];
                            hy.mx = __uint_as_float(opaque_vgpr(__float_as_uint(k == 0 ? v : fmaxf(hy.mx, v))));
                        }
                    if (T == 1 && more) {
#pragma unroll
                        for (int k = 0; k < NC; ++k) {
                            if (N / 2 + k * N / 4 / NC == i) put_k(b2, k);
                            if (3 * N / 4 + k * N / 4 / NC == i) put_v(buf ^ 1, ci + 1, k);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                hy.mx = fmaxf(hy.mx, kvp_other(hy.mx));
                if (has_nan) {
                    // A row's tokens lie in two lanes, hi's eight of every 16; register r of acc[i] is channel 32 i + 8 (r / 4) + 4 hi + r % 4.
                    const uint32_t map = opaque_vgpr(lds_addr(nan_map[buf][4 * hi])) + 4 * T;
                    const uint32_t other = (uint32_t)__shfl_xor((int)hx.seen, 32), a0 = hi ? other : hx.seen, a1 = hi ? hx.seen : other;
                    const uint32_t sees = (a0 & 255u) | ((a1 & 255u) << 8) | ((a0 >> 8) << 16) | ((a1 >> 8) << 24);
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            acc[i][e] = mx_lds4(map + (32 * i + 8 * (e >> 2) + (e & 3)) * 8) & sees ? NAN : acc[i][e];
                }
            };
            half(std::integral_constant<int, 0>{}, sa, ha, sb, hb);
            if constexpr (KB == 2) lds_barrier();
            half(std::integral_constant<int, 1>{}, sb, hb, sa, ha);
        } else {
            if (seen_by_wave(ci + 1)) scores(ci + 1, b1, kb_now, sa, ha);
            first_operands(b1);
            if constexpr (KB == 2) lds_barrier();
            if (more)
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    put_k(b2, i);
                    put_v(buf ^ 1, ci + 1, i);
                }
        }
        kb_piece = kb_now;
        kb_now = bytes();
        const int b = b0;
        b0 = b1;
        b1 = b2;
        b2 = KB == 3 ? b : b0;
    }
    if (!rows_here) return;
    // The lane again, counted: with D = 256 a register that is kept over the loop for it is spilled.
    const int end_lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), end_hi = end_lane >> 5;
    bool k_nan = false, v_nan = false;
    if (__any(largest == 255u)) {
        // A page's scale is NaN.  What the loop made of rows that see one does not matter: they are found here, as
        // branches for them in the loop, or NaN factors, cost 2 to 6%.
        for (int t = c0 * KVD_STEP; t < min(c1 * KVD_STEP, R.ctx); t += 16) {
            const int id = kv8_page(a.batch, c.P, page_log, R.b, t);
            const bool sees = id >= 0 && t < see_hi && t + 16 > see_lo;
            const int64_t scale = (int64_t)max(id, 0) * c.H + h;
            k_nan |= sees && c.ks[scale] == 255;
            v_nan |= sees && c.vs[scale] == 255;
        }
        if (k_nan) l = NAN;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][e] = k_nan | v_nan ? NAN : acc[i][e];
    }
    const int unit = -rest - 127;                        // the accumulators' exponent
    const int row = KVP_WAVE_ROWS * wave + (end_lane & 31);
    l += kvp_other(l);
    const int at_r = R.r0 + row;
    if (at_r >= R.rows) return;
    if (parts > 1) {
        const int64_t at = (((int64_t)tile * c.H + h) * p.splits + split) * ROWS + row;
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
