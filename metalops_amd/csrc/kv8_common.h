// Shared parts of the kernels over the 8-bit key/value cache (kv8_*.hip).
//
// Pages of `page` tokens (a power of two, 16..256).  Keys are held token by token,
// k[P][H][page][D]; values channel by channel, v[P][H][D][page], so that both operands of the
// attention's products are 16-byte loads along the axis that is summed over.  A code is e4m3
// (OCP: 448 the largest, 0x7F NaN, no infinity); scale bytes ks[P][H], vs[P][H] stand for
// 2^(byte - 127).  Sequence b's token t is slot t % page of page table[b][t / page].
#pragma once

#include "mx_common.h"

namespace mcq4 {

struct Kv8Cache {
    uint8_t *k, *v, *ks, *vs;
    int64_t P;
    int H, D, page_log;
    __host__ __device__ int page() const { return 1 << page_log; }
};

// The block table and how the new tokens are dealt out: cu[b] .. cu[b + 1] are sequence b's, or
// `each` to every sequence without cu.
struct Kv8Batch {
    const int32_t *table;
    int64_t table_stride;
    int B, W;
    const int32_t *lens;      // append: tokens before the new ones; read, attention: the context
    const int32_t *cu;
    int each, T;
};

struct Kv8Span { int first, n; };   // a sequence's new tokens
__device__ __forceinline__ Kv8Span kv8_span(const Kv8Batch &t, int b) {
    if (!t.cu) return {b * t.each, t.each};
    // Offsets that do not rise or leave [0, T] count as no tokens.
    const int lo = t.cu[b], hi = t.cu[b + 1];
    if (lo < 0 || hi < lo || hi > t.T) return {0, 0};
    return {lo, hi - lo};
}

// The page of token t of sequence b, or -1: outside the table or not a page of the cache.
__device__ __forceinline__ int kv8_page(const Kv8Batch &t, int64_t P, int page_log, int b, int token) {
    const int j = token >> page_log;
    if (token < 0 || j >= t.W) return -1;
    const int id = t.table[b * t.table_stride + j];
    return (uint32_t)id < (uint64_t)P ? id : -1;
}

// The table's entry for a token of a context that the table covers, unchecked (from the context's
// end on: some entry), and the page that it names.  Apart, so that a load stays in flight until
// its entry is used.
__device__ __forceinline__ int kv8_entry(const Kv8Batch &t, int page_log, int b, int token) {
    return t.table[b * t.table_stride + min(token >> page_log, t.W - 1)];
}
__device__ __forceinline__ int kv8_checked(int entry, int64_t P, int token, int ctx) {
    return ((token < ctx) & ((uint32_t)entry < (uint64_t)P)) ? entry : -1;
}

// Item `item` of a list in which sequence b has count(b) entries: its sequence and its place
// there.  Every lane of the wave takes part; b = B where the list is shorter.
struct Kv8Item { int b, i; };
template <typename F>
__device__ __forceinline__ Kv8Item kv8_locate(int item, int B, F count) {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int own = b0 + lane < B ? count(b0 + lane) : 0;
        int sum = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(sum, d);
            if (lane >= d) sum += up;
        }
        const uint64_t past = __ballot(sum > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            return {b0 + l, item - (__shfl(sum, l) - __shfl(own, l))};
        }
        item -= __shfl(sum, 63);
    }
    return {B, 0};
}

struct Kv8Tokens {                 // k or v of the new tokens, [T][H][D]
    const void *p;
    int64_t token, head;           // strides in elements; channels are neighbours
};

// What the rows of q made of a prefix that their sequences share (kv8_shared.hip): records of `rows` rows, [records][rows][D]
// unnormalised sums and [records][rows][2] maxima and sums of weights, and for each row of q, [T][H G], where they are:
// {the first part's row among all records' rows, parts}, every further part a record on.
struct Kv8Prefix {
    int2 *at;                      // null: no prefix
    float *acc, *ml;
    int2 *own_at;                  // the same of their own tokens, or null
    float *own_acc, *own_ml;
    int rows, own_rows;
    int64_t records, own_records;
    int cost;                      // a piece of a prefix's tile of 128 rows, in pieces of tiles of 16
};

struct Kv8Attend {
    Kv8Cache cache;
    Kv8Batch batch;
    const void *q;
    int64_t q_token, q_head;
    void *out;                     // [T][H G][D]
    float *lse;                    // [T][H G] or null
    int q_dt, G;
    float scale;
    int causal, window;
    int max_context;
    Kv8Prefix pre;
};

// Prefixes s of the sequences groups[s] .. groups[s + 1] - 1 of a batch, or B / S to each without groups.
struct Kv8Shared {
    const int32_t *table;          // [S][stride]
    int64_t stride;
    int S, W;
    const int32_t *lens, *groups;
    int max_prefix;
};
// Whether launch_kv8_shared does all of it; if not it leaves the prefixes' part in a.pre, and launch_kv8_attend does the rest.
bool kv8_shared_own(const Kv8Attend &a, const Kv8Shared &x);
size_t kv8_shared_bytes(const Kv8Attend &a, const Kv8Shared &x, Kv8Prefix *out, void *ws);
hipError_t launch_kv8_shared(const Kv8Attend &a, const Kv8Shared &x, hipStream_t s);

hipError_t launch_kv8_append(const Kv8Cache &c, const Kv8Batch &b, const Kv8Tokens &k, const Kv8Tokens &v, int dt, hipStream_t s);
hipError_t launch_kv8_read(const Kv8Cache &c, const Kv8Batch &b, void *k, void *v, int dt, hipStream_t s);
size_t kv8_attend_workspace_bytes(const Kv8Attend &a);
hipError_t launch_kv8_attend(const Kv8Attend &a, void *ws, hipStream_t s);

}  // namespace mcq4
