// Shared parts of the attention kernels over the 8-bit cache.
#pragma once

#include "kv8_common.h"
#include "mx_gemm.h"

namespace mcq4 {

constexpr int KVD_STEP = 64;                   // tokens taken at a time
constexpr float LOG2E = 1.4426950408889634f;

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
// Times 2^e, any e.
struct Kv8Power {
    float f;
    int e;
    __device__ __forceinline__ explicit Kv8Power(float x) : f(__builtin_amdgcn_exp2f(x - floorf(x))), e((int)floorf(x)) {}
    __device__ __forceinline__ float operator*(float x) const { return __builtin_ldexpf(x * f, e); }
    __device__ __forceinline__ float4_t operator*(float4_t x) const { return float4_t{*this * x[0], *this * x[1], *this * x[2], *this * x[3]}; }
};
// The weights of a row.  A token's score s (a logarithm to base 2) and the scale byte v of its page's values make the
// weight 2^(s + v - m - k + log), in fp16, that multiplies the values' codes, which fp16 holds exactly.  m is the row's
// largest score, l = sum 2^(s - m); k is the largest of the row's s - m + v, a token's part in the output, rounded up,
// so that the weights' largest stands at 2^log: what a row sees alone decides how it is rounded.  (With m as a whole
// number too the largest weight, a power of two so, is rounded: outputs were off by a third more.)
// Where v is so far below k that the values count for nothing, the weight stays at 2^(s - m + KV8_LEAST), 0 in fp16,
// from which l still has its part.
// Scores from KV8_HUGE on come in steps of 1 or more, to which m - log is rounded too, so that weights could pass
// fp16's range.  The kernel of few rows takes m from them first, as they are; that of prompts, where this costs
// 4%, has k leave room for the steps: it holds for scores below 2^30.
constexpr float KV8_NO_K = 1000.f;       // k of a row that has seen nothing
constexpr float KV8_HUGE = 0x1p23f;
constexpr float KV8_LEAST = -80.f;
// k from the largest part, before it is rounded up.
__device__ __forceinline__ float kv8_k(float part) { return part == -INFINITY ? KV8_NO_K : fmaxf(part, -KV8_NO_K); }
// 0xFF in every byte whose code is NaN (0x7F, 0xFF).
__device__ __forceinline__ uint32_t kv8_nan_bytes(uint32_t w) {
    const uint32_t t = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    return (t >> 7) * 0xFFu;
}
__device__ __forceinline__ float kv8_group_max(float x) {      // over the four lanes l % 16 + 16 g
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
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

__device__ __forceinline__ int kv8_same(int v) { return __builtin_amdgcn_readfirstlane(v); }
// The same in every lane, for the compiler's sake.
__device__ __forceinline__ void kv8_uniform(Kv8Rows &R) {
    R = {kv8_same(R.b), kv8_same(R.r0), kv8_same(R.rows), kv8_same(R.first_token), kv8_same(R.ctx), kv8_same(R.pos0), kv8_same(R.lo), kv8_same(R.hi)};
}

// Rows of q that are no sequence's (before the first offset, from the last one on, of a sequence whose offsets count as
// none): 0, their lse -inf.  Every workgroup of `wgs` takes part.  Offsets from 0 to T that rise leave none.
__device__ __forceinline__ void kv8_rest(const Kv8Attend &a, int wg, int wgs) {
    const Kv8Batch &t = a.batch;
    if (!t.cu) return;
    const int lo = t.cu[0], hi = t.cu[t.B];
    if (lo == 0 && hi == t.T) return;
    const bool inside = 0 <= lo && lo <= hi && hi <= t.T;
    const int tid = threadIdx.x, lane = tid & 63, heads = a.cache.H * a.G, pieces = heads * a.cache.D / 8;
    for (int tok = wg; tok < t.T; tok += wgs) {
        if (inside && tok >= lo && tok < hi) continue;
        bool has = false;
        for (int b = lane; b < t.B; b += 64) {
            const Kv8Span sp = kv8_span(t, b);
            has |= tok >= sp.first && tok - sp.first < sp.n;
        }
        if (__any(has)) continue;
        for (int i = tid; i < pieces; i += blockDim.x) *((uint4_t *)a.out + (int64_t)tok * pieces + i) = uint4_t{0, 0, 0, 0};
        if (a.lse)
            for (int i = tid; i < heads; i += blockDim.x) a.lse[(int64_t)tok * heads + i] = -INFINITY;
    }
}

// Tile i of sequence b; false where the sequence has no such row.
__device__ __forceinline__ bool kv8_tile(const Kv8Attend &a, int b, int i, int tile_rows, Kv8Rows &o) {
    const Kv8Span sp = kv8_span(a.batch, b);
    o.b = b;
    o.r0 = i * tile_rows;
    o.rows = sp.n * a.G;
    o.first_token = sp.first;
    if (o.r0 >= o.rows) return false;
    const int most = a.batch.W << a.cache.page_log;
    o.ctx = min(max(a.batch.lens[b], 0), most);
    // A context that holds fewer tokens than are new: the first of them stand before it and see nothing.
    o.pos0 = o.ctx - sp.n;
    const int last = (min(o.r0 + tile_rows, o.rows) - 1) / a.G;
    const int end = a.causal ? min(max(o.pos0 + last + 1, 0), o.ctx) : o.ctx;
    const int begin = a.window ? max(o.pos0 + o.r0 / a.G - a.window + 1, 0) : 0;
    o.lo = begin / KVD_STEP;
    o.hi = end > begin ? (end + KVD_STEP - 1) / KVD_STEP : o.lo;
    return true;
}
// Tile `tile` of `tile_rows` rows where the sequences with the longest contexts come first, each with its
// last (causal: longest) tile first; of more than 64 sequences in the order given.
__device__ __forceinline__ bool kv8_longest_first(const Kv8Attend &a, int tile, int tile_rows, Kv8Rows &o) {
    const int B = a.batch.B, lane = threadIdx.x & 63;
    auto tiles_of = [&](int b) { return (kv8_span(a.batch, b).n * a.G + tile_rows - 1) / tile_rows; };
    int b, i, n;
    if (B <= 64) {
        const int ctx = lane < B ? a.batch.lens[lane] : 0, own = lane < B ? tiles_of(lane) : 0;
        int rank = 0;
        for (int j = 0; j < B; ++j) {
            const int other = __builtin_amdgcn_readlane(ctx, j);
            rank += other > ctx || (other == ctx && j < lane) ? 1 : 0;
        }
        if (lane >= B) rank = lane;
        // To the lane of its rank.
        const int seq = __builtin_amdgcn_ds_permute(rank << 2, lane), count = __builtin_amdgcn_ds_permute(rank << 2, own);
        int sum = count;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(sum, d);
            if (lane >= d) sum += up;
        }
        const uint64_t past = __ballot(sum > tile);
        if (!past) return false;
        const int l = __builtin_ctzll(past);
        b = __builtin_amdgcn_readlane(seq, l);
        n = __builtin_amdgcn_readlane(count, l);
        i = tile - (__builtin_amdgcn_readlane(sum, l) - n);
    } else {
        const Kv8Item it = kv8_locate(tile, B, tiles_of);
        if (it.b >= B) return false;
        b = it.b;
        i = it.i;
        n = tiles_of(b);
    }
    return kv8_tile(a, b, n - 1 - i, tile_rows, o);
}

// How the work is dealt out.  Tiles of 256 or 128 rows (kv8_prefill.hip): a tile's context in parts of
// `span` pieces of 64 tokens.  Tiles of 16 rows (kv8_attend.hip): see there.  A part's record:
// its rows' unnormalised sums, and their maximum and sum of weights.
constexpr int KVD_ROWS = 16;
inline int kvp_rows(int D) { return D <= 128 ? 256 : 128; }
struct Kv8Plan {
    int rows;            // KVD_ROWS or kvp_rows
    int tiles;           // upper bound over all sequences
    int splits, span;    // large tiles: most parts of a tile, and their pieces
    int wgs, chunk;      // 16 rows: workgroups, and least pieces of one (0: by the average context)
    int records;
    float *acc;          // [records][rows][D]
    float *ml;           // [records][rows][2]
    uint32_t *tickets;   // 16 rows: [wgs], 0 before and after
};
__device__ __forceinline__ int kv8_parts(const Kv8Rows &R, const Kv8Plan &p) {
    return max(1, min(p.splits, (R.hi - R.lo + p.span - 1) / p.span));
}
hipError_t launch_kv8_decode(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s);
hipError_t launch_kv8_prefill(const Kv8Attend &a, const Kv8Plan &p, hipStream_t s);

}  // namespace mcq4
