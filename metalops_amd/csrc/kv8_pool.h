// Pages that the layers' caches share (kv8_pool.hip).
#pragma once

#include "kv8_common.h"

namespace mcq4 {

struct Kv8Pool {
    uint8_t *const *tensors;       // device, [layers][4]: a cache's k, v, ks, vs
    int32_t *refs;                 // [P]
    int64_t P;
    int layers, H, D, page_log;
};
struct Kv8Fork {
    const int32_t *table;          // [B][stride]
    int64_t stride;
    const int32_t *lens, *parents; // [B], [rows]
    int32_t *out, *out_lens;       // [rows][W], [rows]
    int B, W, rows, release;
};
struct Kv8Resize {
    int32_t *table;
    int64_t stride;
    const int32_t *lens, *new_lens;
    int32_t *missing;
    int B, W;
};
struct Kv8List { int32_t *count, *src, *dst; };

hipError_t launch_kv8_copy_pages(const Kv8Pool &p, const int32_t *src, const int32_t *dst, int64_t n, hipStream_t s);
hipError_t launch_kv8_fork(const Kv8Pool &p, const Kv8Fork &f, hipStream_t s);
size_t kv8_resize_bytes(const Kv8Pool &p, int64_t B);
hipError_t launch_kv8_resize(const Kv8Pool &p, const Kv8Resize &r, void *ws, hipStream_t s);
size_t kv8_compact_bytes(const Kv8Pool &p);
hipError_t launch_kv8_compact(const Kv8Pool &p, int32_t *names, int32_t *live, void *ws, hipStream_t s);
hipError_t launch_kv8_rename(int32_t *table, int64_t stride, int64_t B, int W, const int32_t *names, int64_t P, hipStream_t s);

}  // namespace mcq4
