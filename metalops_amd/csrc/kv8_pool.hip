// Pages of the 8-bit cache dealt out, shared, copied and moved together, without the host knowing which.
//
// refs[p] counts the block tables' entries that name page p; 0: the page is free.  All layers' caches share
// page numbers, so a page is copied in each of them.  Decisions are a prefix sum over the sequences or over
// refs, made by one workgroup (refs of 2048 pages are 8 KB: one round trip), which leaves a list of pages to
// copy; the copy is a launch of its own over the whole card.  Every rule picks lowest numbers first, so that
// results do not depend on the order in which anything runs.
#include <algorithm>

#include "kv8_common.h"
#include "kv8_pool.h"

namespace mcq4 {

constexpr int KVL_THREADS = 1024, KVL_WAVES = KVL_THREADS / 64;

// What precedes a thread's `x` in the workgroup, and the workgroup's sum.  Two 32-bit counts at a time.
struct Kv8Sum { uint64_t before, all; };
__device__ __forceinline__ Kv8Sum kv8_scan(uint64_t x, uint64_t *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    __syncthreads();                               // lds has been read
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < KVL_WAVES; ++w) {
        const uint64_t v = lds[w];
        if (w < wave) before += v;
        all += v;
    }
    return {before + sum - x, all};
}
__device__ __forceinline__ uint64_t kv8_two(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }

// refs is changed by atomics, at the L2, and read past the L1.
__device__ __forceinline__ int kv8_refs(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void kv8_add(int32_t *p, int by) { __hip_atomic_fetch_add(p, by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__device__ __forceinline__ int kv8_tokens(int n, int W, int page_log) { return min(max(n, 0), W << page_log); }
__device__ __forceinline__ int kv8_pages(int tokens, int page_log) { return (tokens >> page_log) + ((tokens & ((1 << page_log) - 1)) != 0); }

// ---- fork ----

// Workgroup i < rows makes row i of the new table; the others change the counts of an old row's pages, by the
// rows that it became.
__global__ void __launch_bounds__(256)
kv8_fork_kernel(Kv8Pool p, Kv8Fork f) {
    const int wg = blockIdx.x, tid = threadIdx.x;
    if (wg < f.rows) {
        const int from = f.parents[wg];
        const bool ok = (uint32_t)from < (uint32_t)f.B;
        const int n = ok ? kv8_tokens(f.lens[from], f.W, p.page_log) : 0, used = kv8_pages(n, p.page_log);
        for (int j = tid; j < f.W; j += 256) f.out[(int64_t)wg * f.W + j] = j < used ? f.table[from * f.stride + j] : -1;
        if (tid == 0) f.out_lens[wg] = n;
        return;
    }
    const int b = wg - f.rows;
    __shared__ int became;
    if (tid == 0) became = 0;
    __syncthreads();
    int mine = 0;
    for (int i = tid; i < f.rows; i += 256) mine += f.parents[i] == b;
    if (mine) atomicAdd(&became, mine);
    __syncthreads();
    const int by = became - f.release;
    if (by == 0) return;
    const int used = kv8_pages(kv8_tokens(f.lens[b], f.W, p.page_log), p.page_log);
    for (int j = tid; j < used; j += 256) {
        const int id = f.table[b * f.stride + j];
        if ((uint32_t)id < (uint64_t)p.P) kv8_add(p.refs + id, by);
    }
}

// ---- resize ----

constexpr int KVL_EACH = 8, KVL_TILE = KVL_THREADS * KVL_EACH;      // refs looked at at a time
// A row's entries are a thread's work where there are no more of them, else a wave's.  Two calls, rows that get pages and give
// them back, by threads and by waves: 256 rows of one page 22 and 42 us, 2048 of one 30 and 186, 1024 of four 30 and 106, 256 of
// eight 27.5 and 41.5, 64 of sixteen 31.2 and 26.2.
constexpr int KVL_FEW = 8;
// The counts of pages p0 + 8 tid .. of a tile; pages past the last one are in use.
struct Kv8Counts { int n[KVL_EACH]; };
__device__ __forceinline__ Kv8Counts kv8_counts(const Kv8Pool &p, int64_t p0) {
    Kv8Counts c;
#pragma unroll
    for (int e = 0; e < KVL_EACH; ++e) {
        const int64_t id = p0 + (int64_t)threadIdx.x * KVL_EACH + e;
        c.n[e] = id < p.P ? kv8_refs(p.refs + id) : 1;
    }
    return c;
}

struct Kv8Grow { int old_pages, new_pages, tokens, grows; };
__device__ __forceinline__ Kv8Grow kv8_grow(const Kv8Pool &p, const Kv8Resize &r, int b) {
    const int was = kv8_tokens(r.lens[b], r.W, p.page_log), now = kv8_tokens(r.new_lens[b], r.W, p.page_log);
    return {kv8_pages(was, p.page_log), kv8_pages(now, p.page_log), was, now > was};
}

// ws: at[B] (a row's first new page in the list), given[P] and the copies src[B], dst[B], count.
//
// A chain of round trips to memory by one workgroup, each a microsecond: lengths and counts together, the last pages
// of rows that grow, their counts, then what is dealt out.  The workgroup's barriers order its own accesses (counts are
// changed and read past the L1); device-wide fences between the steps made 13.5 us of 8.
__global__ void __launch_bounds__(KVL_THREADS)
kv8_resize_kernel(Kv8Pool p, Kv8Resize r, Kv8List list, int32_t *at, int32_t *given) {
    __shared__ uint64_t lds[KVL_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Kv8Counts first = kv8_counts(p, 0);            // on their way meanwhile
    // What sequences give back, first.
    int gives = 0;                                 // the most of a row
    for (int b = tid; b < r.B; b += KVL_THREADS) {
        const Kv8Grow g = kv8_grow(p, r, b);
        gives = max(gives, g.old_pages - g.new_pages);
    }
    if (__syncthreads_or(gives > 0)) {
        const bool many = __syncthreads_or(gives > KVL_FEW);
        for (int b = many ? wave : tid; b < r.B; b += many ? KVL_WAVES : KVL_THREADS) {
            const Kv8Grow g = kv8_grow(p, r, b);
            int32_t *row = r.table + b * r.stride;
            for (int j = g.new_pages + (many ? lane : 0); j < g.old_pages; j += many ? 64 : 1) {
                const int id = row[j];
                if ((uint32_t)id < (uint64_t)p.P) {
                    kv8_add(p.refs + id, -1);
                    row[j] = -1;
                }
            }
        }
        __syncthreads();
        first = kv8_counts(p, 0);
    }
    // How many pages each needs; bit 31 of at: it copies its last one.
    uint32_t pages = 0, copies = 0;
    for (int b0 = 0; b0 < r.B; b0 += KVL_THREADS) {
        const int b = b0 + tid;
        uint32_t n = 0, copy = 0;
        if (b < r.B) {
            const Kv8Grow g = kv8_grow(p, r, b);
            if (g.grows && (g.tokens & ((1 << p.page_log) - 1))) {
                const int id = r.table[b * r.stride + g.old_pages - 1];
                copy = (uint32_t)id < (uint64_t)p.P && kv8_refs(p.refs + id) > 1;
            }
            n = copy + max(g.new_pages - g.old_pages, 0);
        }
        const Kv8Sum s = kv8_scan(kv8_two(n, copy), lds);
        if (b < r.B) {
            at[b] = (int32_t)((pages + (uint32_t)s.before) | copy << 31);
            if (copy) list.src[copies + (uint32_t)(s.before >> 32)] = b;         // the row, for now
        }
        pages += (uint32_t)s.all;
        copies += (uint32_t)(s.all >> 32);
    }
    // The first free pages, in order, as many as are needed.
    uint32_t found = 0;
    for (int64_t p0 = 0; p0 < p.P && found < pages; p0 += KVL_TILE) {
        if (p0 > 0) first = kv8_counts(p, p0);
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < KVL_EACH; ++e) n += first.n[e] <= 0;
        const Kv8Sum s = kv8_scan(n, lds);
        uint32_t place = found + (uint32_t)s.before;
#pragma unroll
        for (int e = 0; e < KVL_EACH; ++e)
            if (first.n[e] <= 0) {
                if (place < pages) given[place] = (int32_t)(p0 + (int64_t)tid * KVL_EACH + e);
                ++place;
            }
        found += (uint32_t)s.all;
    }
    const uint32_t missing = pages > found ? pages - found : 0;
    if (tid == 0) {
        *r.missing = (int32_t)missing;
        *list.count = missing ? 0 : (int32_t)copies;
    }
    if (missing || !pages) return;
    __syncthreads();
    for (uint32_t i = tid; i < copies; i += KVL_THREADS) {
        const int b = list.src[i], to = given[at[b] & 0x7FFFFFFF];
        int32_t *entry = r.table + b * r.stride + kv8_grow(p, r, b).old_pages - 1;
        const int from = *entry;
        list.src[i] = from;
        list.dst[i] = to;
        *entry = to;
        kv8_add(p.refs + from, -1);
        p.refs[to] = 1;
    }
    const bool few = pages <= KVL_FEW * (uint32_t)r.B;
    for (int b = few ? tid : wave; b < r.B; b += few ? KVL_THREADS : KVL_WAVES) {
        const Kv8Grow g = kv8_grow(p, r, b);
        const uint32_t a = (uint32_t)at[b], start = (a & 0x7FFFFFFFu) + (a >> 31);
        for (int j = g.old_pages + (few ? 0 : lane); j < g.new_pages; j += few ? 1 : 64) {
            const int id = given[start + (j - g.old_pages)];
            r.table[b * r.stride + j] = id;
            p.refs[id] = 1;
        }
    }
}

// ---- compact ----

__global__ void __launch_bounds__(KVL_THREADS)
kv8_compact_kernel(Kv8Pool p, Kv8List list, int32_t *names, int32_t *live) {
    __shared__ uint64_t lds[KVL_WAVES];
    const int tid = threadIdx.x;
    Kv8Counts c = kv8_counts(p, 0);
    uint32_t n = 0;
    for (int64_t p0 = 0; p0 < p.P; p0 += KVL_TILE) {
        if (p0 > 0) c = kv8_counts(p, p0);
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < KVL_EACH; ++e) mine += c.n[e] > 0 && p0 + (int64_t)tid * KVL_EACH + e < p.P;
        n += (uint32_t)kv8_scan(mine, lds).all;
#pragma unroll
        for (int e = 0; e < KVL_EACH; ++e) {
            const int64_t id = p0 + e * KVL_THREADS + tid;
            if (id < p.P) names[id] = (int32_t)id;
        }
    }
    // Pages in use behind the first n, and free ones among them: as many.  Both are listed in order.
    uint32_t moved = 0, holes = 0;
    for (int64_t p0 = 0; p0 < p.P; p0 += KVL_TILE) {
        if (p.P > KVL_TILE) c = kv8_counts(p, p0);
        uint32_t m = 0, f = 0;
#pragma unroll
        for (int e = 0; e < KVL_EACH; ++e) {
            const int64_t id = p0 + (int64_t)tid * KVL_EACH + e;
            m += id < p.P && id >= n && c.n[e] > 0;
            f += id < n && c.n[e] <= 0;
        }
        const Kv8Sum s = kv8_scan(kv8_two(m, f), lds);
        uint32_t at_m = moved + (uint32_t)s.before, at_f = holes + (uint32_t)(s.before >> 32);
#pragma unroll
        for (int e = 0; e < KVL_EACH; ++e) {
            const int64_t id = p0 + (int64_t)tid * KVL_EACH + e;
            if (id < p.P && id >= n && c.n[e] > 0) list.src[at_m++] = (int32_t)id;
            if (id < n && c.n[e] <= 0) list.dst[at_f++] = (int32_t)id;
        }
        moved += (uint32_t)s.all;
        holes += (uint32_t)(s.all >> 32);
    }
    if (tid == 0) {
        *live = (int32_t)n;
        *list.count = (int32_t)moved;
    }
    __syncthreads();
    for (uint32_t i = tid; i < moved; i += KVL_THREADS) {
        const int from = list.src[i], to = list.dst[i];
        names[from] = to;
        p.refs[to] = kv8_refs(p.refs + from);
        p.refs[from] = 0;
    }
}

__global__ void __launch_bounds__(256)
kv8_rename_kernel(int32_t *table, int64_t stride, int W, int64_t entries, const int32_t *names, int64_t P) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= entries) return;
    int32_t *entry = table + i / W * stride + i % W;
    const int id = *entry;
    if ((uint32_t)id < (uint64_t)P) *entry = names[id];
}

// ---- copies ----

// A workgroup takes 16 KB of a page's keys and values in a layer at a time, four loads of 16 bytes a thread in
// flight.  count: of the list, on the device, or null for `most`.  What is written is not read soon, so it goes past the
// caches; what is read does too where no page is in the list twice (ONCE), as when pages are moved: 500 pages of four layers,
// 8 heads of 64 x 128, take 106 us in all (520 MB; 120 with ordinary accesses of 32 KB, 112 with ordinary loads), while copies of
// one page for many rows take 46 us with such loads and 40 without.
constexpr int KVC_EACH = 4;
template <bool ONCE>
__global__ void __launch_bounds__(256)
kv8_copy_kernel(Kv8Pool p, const int32_t *src, const int32_t *dst, const int32_t *count, int most, int chunks) {
    const int64_t n = count ? *count : most, items = n * p.layers * chunks;
    const int tid = threadIdx.x;
    const uint32_t page16 = (uint32_t)((int64_t)p.H * p.D * (1 << p.page_log) / 16);      // of K, and of V
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int chunk = (int)(item % chunks), layer = (int)(item / chunks % p.layers);
        const int64_t i = item / chunks / p.layers;
        const int from = src[i], to = dst[i];
        if ((uint32_t)from >= (uint64_t)p.P || (uint32_t)to >= (uint64_t)p.P) continue;
        uint8_t *const *t = p.tensors + 4 * layer;
        uint4_t *const k = (uint4_t *)t[0], *const v = (uint4_t *)t[1];
        uint4_t x[KVC_EACH];
#pragma unroll
        for (int e = 0; e < KVC_EACH; ++e) {
            const uint32_t u = (chunk * KVC_EACH + e) * 256 + tid;
            const uint4_t *const at = u < page16 ? k + (int64_t)from * page16 + u : v + (int64_t)from * page16 + u - page16;
            if (u < 2 * page16) x[e] = ONCE ? __builtin_nontemporal_load(at) : *at;
        }
#pragma unroll
        for (int e = 0; e < KVC_EACH; ++e) {
            const uint32_t u = (chunk * KVC_EACH + e) * 256 + tid;
            uint4_t *const at = u < page16 ? k + (int64_t)to * page16 + u : v + (int64_t)to * page16 + u - page16;
            if (u < 2 * page16) __builtin_nontemporal_store(x[e], at);
        }
        if (chunk == 0)
            for (int h = tid; h < 2 * p.H; h += 256) {
                uint8_t *const s = h < p.H ? t[2] : t[3];
                const int hh = h < p.H ? h : h - p.H;
                s[(int64_t)to * p.H + hh] = s[(int64_t)from * p.H + hh];
            }
    }
}

// As many workgroups as the list may need, up to a number whose start costs little where it turns out empty (16384: 2 us
// more than 4096, and 4 us less where 500 pages move; 65536 cost 12).
template <bool ONCE>
static hipError_t launch_kv8_copies(const Kv8Pool &p, const int32_t *src, const int32_t *dst, const int32_t *count, int64_t most, hipStream_t s) {
    const int64_t units = 2 * ((int64_t)p.H * p.D * (1 << p.page_log) / 16);
    const int chunks = (int)((units + 256 * KVC_EACH - 1) / (256 * KVC_EACH));
    const int64_t items = most * p.layers * chunks;
    if (!items) return hipSuccess;
    hipLaunchKernelGGL(kv8_copy_kernel<ONCE>, dim3((unsigned)std::min<int64_t>(items, ONCE ? 16384 : 4096)), dim3(256), 0, s, p, src, dst, count, (int)most, chunks);
    return hipGetLastError();
}

hipError_t launch_kv8_copy_pages(const Kv8Pool &p, const int32_t *src, const int32_t *dst, int64_t n, hipStream_t s) {
    return launch_kv8_copies<false>(p, src, dst, nullptr, n, s);
}

hipError_t launch_kv8_fork(const Kv8Pool &p, const Kv8Fork &f, hipStream_t s) {
    hipLaunchKernelGGL(kv8_fork_kernel, dim3((unsigned)(f.rows + f.B)), dim3(256), 0, s, p, f);
    return hipGetLastError();
}

size_t kv8_resize_bytes(const Kv8Pool &p, int64_t B) { return ((size_t)3 * B + (size_t)p.P + 1) * sizeof(int32_t); }
hipError_t launch_kv8_resize(const Kv8Pool &p, const Kv8Resize &r, void *ws, hipStream_t s) {
    int32_t *w = (int32_t *)ws;
    const Kv8List list = {w, w + 1, w + 1 + r.B};
    hipLaunchKernelGGL(kv8_resize_kernel, dim3(1), dim3(KVL_THREADS), 0, s, p, r, list, w + 1 + 2 * (int64_t)r.B, w + 1 + 3 * (int64_t)r.B);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_kv8_copies<false>(p, list.src, list.dst, list.count, r.B, s);
}

size_t kv8_compact_bytes(const Kv8Pool &p) { return ((size_t)2 * p.P + 1) * sizeof(int32_t); }
hipError_t launch_kv8_compact(const Kv8Pool &p, int32_t *names, int32_t *live, void *ws, hipStream_t s) {
    int32_t *w = (int32_t *)ws;
    const Kv8List list = {w, w + 1, w + 1 + p.P};
    hipLaunchKernelGGL(kv8_compact_kernel, dim3(1), dim3(KVL_THREADS), 0, s, p, list, names, live);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_kv8_copies<true>(p, list.src, list.dst, list.count, p.P / 2, s);
}

hipError_t launch_kv8_rename(int32_t *table, int64_t stride, int64_t B, int W, const int32_t *names, int64_t P, hipStream_t s) {
    const int64_t entries = B * W;
    hipLaunchKernelGGL(kv8_rename_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, s, table, stride, W, entries, names, P);
    return hipGetLastError();
}

}  // namespace mcq4
