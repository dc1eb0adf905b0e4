// C ABI of the microscaled 4-bit products and of the 8-bit key/value cache: argument
// validation, status codes and dispatch.  No allocation, no exceptions; everything is
// enqueued on the caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <utility>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/mcq4.h"
#include "kv8_common.h"
#include "kv8_pool.h"
#include "qk_rope.h"

namespace mcq4 {
int set_error(int code, const char *msg);   // mcq4_capi.cpp
}

namespace {

constexpr int64_t kMaxDim = (int64_t)1 << 30;

int fail(int code, const char *fmt, ...) {
    char msg[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    return mcq4::set_error(code, msg);
}
int hip_status(hipError_t e, const char *what) {
    if (e == hipSuccess) return mcq4::set_error(MCQ4_OK, "");
    return fail(MCQ4_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
// Before a call that changes counts: an error that an earlier one has left would be taken for its own, once it is on its way.
int earlier_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MCQ4_OK : fail(MCQ4_ERR_HIP, "left by an earlier call, nothing enqueued: %s", hipGetErrorString(e));
}
bool aligned(const void *p, uintptr_t a) { return (uintptr_t)p % a == 0; }
bool valid_dt(int dt) { return dt == MCQ4_DTYPE_F32 || dt == MCQ4_DTYPE_F16 || dt == MCQ4_DTYPE_BF16; }
int64_t dt_size(int dt) { return dt == MCQ4_DTYPE_F32 ? 4 : 2; }

// Rows and row length of a microscaled matrix: the conversions count its 8-element pieces in 32 bits.
int check_rows(int64_t R, int64_t K) {
    if (R <= 0 || R > kMaxDim) return fail(MCQ4_ERR_SHAPE, "rows (%lld) out of range", (long long)R);
    if (K <= 0 || K > kMaxDim || K % 32) return fail(MCQ4_ERR_SHAPE, "K (%lld) must be divisible by 32", (long long)K);
    if (R * (K / 8) >= ((int64_t)1 << 32) - 4096) return fail(MCQ4_ERR_SHAPE, "%lld x %lld elements are too many", (long long)R, (long long)K);
    return MCQ4_OK;
}

int matmul_checks(const mcq4::MxCall &c) {
    if (!c.X || !c.W || !c.Ws || !c.Y) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(c.x_dt)) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    if (c.K <= 0 || c.K > kMaxDim || c.K % 32) return fail(MCQ4_ERR_SHAPE, "K (%lld) must be divisible by 32", (long long)c.K);
    if (c.N <= 0 || c.N > kMaxDim) return fail(MCQ4_ERR_SHAPE, "N (%lld) out of range", (long long)c.N);
    if (c.M <= 0 || c.M > (int64_t)1 << 20) return fail(MCQ4_ERR_SHAPE, "M (%lld) out of range", (long long)c.M);
    if (c.ldy < c.N) return fail(MCQ4_ERR_SHAPE, "ldy (%lld) < N (%lld)", (long long)c.ldy, (long long)c.N);
    if (!aligned(c.W, 16)) return fail(MCQ4_ERR_ALIGNMENT, "packed weights must be 16-byte aligned");
    if (!aligned(c.Y, dt_size(c.x_dt))) return fail(MCQ4_ERR_ALIGNMENT, "Y must be aligned to its element size");
    if (!aligned(c.X, 16)) return fail(MCQ4_ERR_ALIGNMENT, "X must be 16-byte aligned");
    if (!c.Xs) {
        if (c.ldx < c.K) return fail(MCQ4_ERR_SHAPE, "ldx (%lld) < K (%lld)", (long long)c.ldx, (long long)c.K);
        if (c.ldx * dt_size(c.x_dt) % 16) return fail(MCQ4_ERR_ALIGNMENT, "X rows must be 16-byte aligned (ldx %lld)", (long long)c.ldx);
    }
    return MCQ4_OK;
}

int matmul(const mcq4::MxCall &c, void *workspace, size_t workspace_bytes, void *stream, const char *what) {
    if (int st = matmul_checks(c)) return st;
    const mcq4::MxPlan plan = mcq4::mx_plan(c);
    const size_t need = mcq4::mx_workspace_bytes(plan);
    if (need && (!workspace || workspace_bytes < need))
        return fail(MCQ4_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (need && !aligned(workspace, 16)) return fail(MCQ4_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    return hip_status(mcq4::launch_mx(c, plan, need ? (char *)workspace + mcq4::COUNTER_BYTES : nullptr, (hipStream_t)stream), what);
}

int check_cache(const mcq4_kv8_cache *c, const mcq4_kv8_batch *b, mcq4::Kv8Cache &co, mcq4::Kv8Batch &bo, bool tokens) {
    if (!c || !b || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !b->block_table || !b->lens)
        return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(MCQ4_ERR_SHAPE, "page_size (%d) must be 16, 32, 64, 128 or 256", c->page_size);
    if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % 16)
        return fail(MCQ4_ERR_SHAPE, "head_dim (%d) must be a multiple of 16 up to 256", c->head_dim);
    if (c->kv_heads <= 0 || c->kv_heads > 65535) return fail(MCQ4_ERR_SHAPE, "kv_heads (%d) out of range", c->kv_heads);
    if (c->num_pages <= 0 || c->num_pages > kMaxDim) return fail(MCQ4_ERR_SHAPE, "num_pages (%lld) out of range", (long long)c->num_pages);
    if ((int64_t)c->kv_heads * c->page_size * c->head_dim >= (int64_t)1 << 31)
        return fail(MCQ4_ERR_SHAPE, "a page of %d heads of %d x %d codes is too large", c->kv_heads, c->page_size, c->head_dim);
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16)) return fail(MCQ4_ERR_ALIGNMENT, "codes must be 16-byte aligned");
    if (b->batch <= 0 || b->batch > 1 << 20) return fail(MCQ4_ERR_SHAPE, "batch (%d) out of range", b->batch);
    if (b->width <= 0 || (int64_t)b->width * c->page_size > kMaxDim)
        return fail(MCQ4_ERR_SHAPE, "block table width (%d) out of range", b->width);
    if (b->batch > 1 && b->table_stride < b->width) return fail(MCQ4_ERR_SHAPE, "table_stride (%lld) < width (%d)", (long long)b->table_stride, b->width);
    if ((int64_t)b->batch * b->width > kMaxDim) return fail(MCQ4_ERR_SHAPE, "block table of %d x %d entries is too large", b->batch, b->width);
    if (!aligned(b->block_table, 4) || !aligned(b->lens, 4) || !aligned(b->cu_seqlens, 4))
        return fail(MCQ4_ERR_ALIGNMENT, "block_table, lens and cu_seqlens must be aligned to 4 bytes");
    if (tokens) {
        if (b->T <= 0 || b->T > 1 << 24) return fail(MCQ4_ERR_SHAPE, "T (%lld) out of range", (long long)b->T);
        if (!b->cu_seqlens && b->T % b->batch)
            return fail(MCQ4_ERR_SHAPE, "T (%lld) must be a multiple of the batch (%d) without cu_seqlens", (long long)b->T, b->batch);
    }
    int log = 4;
    while (1 << log < c->page_size) ++log;
    co = {c->k_codes, c->v_codes, c->k_scales, c->v_scales, c->num_pages, c->kv_heads, c->head_dim, log};
    bo = {b->block_table, b->table_stride, b->batch, b->width, b->lens, b->cu_seqlens, (int)(tokens ? b->T / b->batch : 0), (int)(tokens ? b->T : 0)};
    return MCQ4_OK;
}

int check_prefixes(const mcq4::Kv8Attend &a, const mcq4_kv8_batch *b, const mcq4_kv8_prefixes *p, int32_t heads, int64_t max_prefix,
                   mcq4::Kv8Shared &o) {
    if (!p || !p->block_table || !p->lens) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (p->prefixes <= 0 || p->prefixes > 1 << 20) return fail(MCQ4_ERR_SHAPE, "prefixes (%d) out of range", p->prefixes);
    if (p->width <= 0 || (int64_t)p->width << a.cache.page_log > kMaxDim)
        return fail(MCQ4_ERR_SHAPE, "width of the prefixes' block table (%d) out of range", p->width);
    if (p->prefixes > 1 && p->table_stride < p->width)
        return fail(MCQ4_ERR_SHAPE, "table_stride (%lld) of the prefixes < width (%d)", (long long)p->table_stride, p->width);
    if ((int64_t)p->prefixes * p->width > kMaxDim)
        return fail(MCQ4_ERR_SHAPE, "block table of %d x %d entries is too large", p->prefixes, p->width);
    if (!aligned(p->block_table, 4) || !aligned(p->lens, 4) || !aligned(p->groups, 4))
        return fail(MCQ4_ERR_ALIGNMENT, "block_table, lens and groups of the prefixes must be aligned to 4 bytes");
    if (!p->groups && b->batch % p->prefixes)
        return fail(MCQ4_ERR_SHAPE, "the batch (%d) must be a multiple of the prefixes (%d) without groups", b->batch, p->prefixes);
    if (max_prefix < 0) return fail(MCQ4_ERR_SHAPE, "max_prefix (%lld) is negative", (long long)max_prefix);
    // The pieces of 64 tokens of all tiles are counted in 31 bits.
    const int64_t pieces = (((int64_t)p->width << a.cache.page_log) + 63) / 64 + 8, tiles = b->T * (heads / a.cache.H) / 16 + p->prefixes;
    if (pieces > ((int64_t)1 << 30) / a.cache.H / tiles)
        return fail(MCQ4_ERR_SHAPE, "%lld new tokens behind prefixes of up to %lld are too many", (long long)b->T, (long long)p->width << a.cache.page_log);
    o = {p->block_table, p->table_stride, p->prefixes, p->width, p->lens, p->groups, (int)std::min<int64_t>(max_prefix, kMaxDim)};
    return MCQ4_OK;
}

// The workspace: counters, what the kernels of the sequences' own tokens need where they run, and the prefixes' records,
// whose rows are counted in 31 bits (else 0).
size_t shared_bytes(mcq4::Kv8Attend &a, const mcq4::Kv8Shared &x) {
    const size_t n = mcq4::kv8_shared_bytes(a, x, &a.pre, (void *)16);      // not used but for being there
    if (std::max(a.pre.records * a.pre.rows, a.pre.own_records * a.pre.own_rows) > INT32_MAX) return 0;
    return mcq4::COUNTER_BYTES + n + (mcq4::kv8_shared_own(a, x) ? 0 : mcq4::kv8_attend_workspace_bytes(a));
}

int check_pool(const mcq4_kv8_pool *p, mcq4::Kv8Pool &o) {
    if (!p || !p->tensors || !p->refs) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return fail(MCQ4_ERR_SHAPE, "page_size (%d) must be 16, 32, 64, 128 or 256", p->page_size);
    if (p->head_dim <= 0 || p->head_dim > 256 || p->head_dim % 16)
        return fail(MCQ4_ERR_SHAPE, "head_dim (%d) must be a multiple of 16 up to 256", p->head_dim);
    if (p->kv_heads <= 0 || p->kv_heads > 65535) return fail(MCQ4_ERR_SHAPE, "kv_heads (%d) out of range", p->kv_heads);
    if (p->layers <= 0 || p->layers > 65535) return fail(MCQ4_ERR_SHAPE, "layers (%d) out of range", p->layers);
    if (p->num_pages <= 0 || p->num_pages > kMaxDim) return fail(MCQ4_ERR_SHAPE, "num_pages (%lld) out of range", (long long)p->num_pages);
    if ((int64_t)p->kv_heads * p->page_size * p->head_dim >= (int64_t)1 << 31)
        return fail(MCQ4_ERR_SHAPE, "a page of %d heads of %d x %d codes is too large", p->kv_heads, p->page_size, p->head_dim);
    if (!aligned(p->tensors, 8) || !aligned(p->refs, 4)) return fail(MCQ4_ERR_ALIGNMENT, "tensors must be aligned to 8 bytes, refs to 4");
    int log = 4;
    while (1 << log < p->page_size) ++log;
    o = {p->tensors, p->refs, p->num_pages, p->layers, p->kv_heads, p->head_dim, log};
    return MCQ4_OK;
}

int check_table(const int32_t *table, int64_t stride, int64_t B, int64_t W, int page_log) {
    if (!table) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (B <= 0 || B > 1 << 20) return fail(MCQ4_ERR_SHAPE, "batch (%lld) out of range", (long long)B);
    if (W <= 0 || W > kMaxDim >> page_log) return fail(MCQ4_ERR_SHAPE, "block table width (%lld) out of range", (long long)W);
    if (B > 1 && stride < W) return fail(MCQ4_ERR_SHAPE, "table_stride (%lld) < width (%lld)", (long long)stride, (long long)W);
    if (B * W > kMaxDim) return fail(MCQ4_ERR_SHAPE, "block table of %lld x %lld entries is too large", (long long)B, (long long)W);
    if (!aligned(table, 4)) return fail(MCQ4_ERR_ALIGNMENT, "block_table must be aligned to 4 bytes");
    return MCQ4_OK;
}

int check_heads(const mcq4_kv8_cache *c, const mcq4_kv8_batch *b, int32_t heads, int32_t window, int64_t max_context) {
    if (heads <= 0 || heads > 65535 || heads % c->kv_heads)
        return fail(MCQ4_ERR_SHAPE, "heads (%d) must be a multiple of kv_heads (%d)", heads, c->kv_heads);
    if (window < 0 || window > kMaxDim) return fail(MCQ4_ERR_SHAPE, "window (%d) out of range", window);
    if (max_context < 0) return fail(MCQ4_ERR_SHAPE, "max_context (%lld) is negative", (long long)max_context);
    if (b->T * heads > kMaxDim) return fail(MCQ4_ERR_SHAPE, "%lld tokens of %d heads are too many", (long long)b->T, heads);
    return MCQ4_OK;
}

}  // namespace

extern "C" {

int mcq4_quantize_mxfp4(const void *X, int x_dtype, int64_t row_stride, int64_t col_stride, int64_t R, int64_t K,
                        uint8_t *packed, uint8_t *scales, void *stream) {
    if (!X || !packed || !scales) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(x_dtype)) return fail(MCQ4_ERR_INVALID_ARG, "x_dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    if (int st = check_rows(R, K)) return st;
    if (row_stride < 0 || col_stride < 0) return fail(MCQ4_ERR_SHAPE, "strides must not be negative");
    if ((K / 32 + 7) / 8 > 65535 && col_stride != 1) return fail(MCQ4_ERR_SHAPE, "K (%lld) too large", (long long)K);
    if (!aligned(X, dt_size(x_dtype))) return fail(MCQ4_ERR_ALIGNMENT, "X must be aligned to its element size");
    if (!aligned(packed, 16)) return fail(MCQ4_ERR_ALIGNMENT, "packed must be 16-byte aligned");
    return hip_status(mcq4::launch_mx_quantize(X, x_dtype, row_stride, col_stride, R, K, packed, scales, (hipStream_t)stream),
                      "mxfp4 quantize launch");
}

int mcq4_dequantize_mxfp4(const uint8_t *packed, const uint8_t *scales, int64_t R, int64_t K, void *out, int out_dtype,
                          void *stream) {
    if (!packed || !scales || !out) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(out_dtype)) return fail(MCQ4_ERR_INVALID_ARG, "out_dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    if (int st = check_rows(R, K)) return st;
    if (!aligned(packed, 16) || !aligned(out, 16)) return fail(MCQ4_ERR_ALIGNMENT, "packed and out must be 16-byte aligned");
    return hip_status(mcq4::launch_mx_dequantize(packed, scales, R, K, out, out_dtype, (hipStream_t)stream), "mxfp4 dequantize launch");
}

size_t mcq4_matmul_mxfp4_workspace_bytes(int64_t M, int64_t K, int64_t N, int x_dtype) {
    if (M <= 0 || K <= 0 || N <= 0 || K % 32 || !valid_dt(x_dtype)) return 0;
    mcq4::MxCall c = {};
    c.x_dt = x_dtype; c.M = M; c.K = K; c.N = N;
    return mcq4::mx_workspace_bytes(mcq4::mx_plan(c));
}

int mcq4_matmul_mxfp4(const void *X, int x_dtype, int64_t ldx, const uint8_t *W, const uint8_t *W_scales, void *Y,
                      int64_t ldy, int64_t M, int64_t K, int64_t N, void *workspace, size_t workspace_bytes, void *stream) {
    return matmul({X, nullptr, x_dtype, ldx, W, W_scales, Y, ldy, M, K, N, nullptr}, workspace, workspace_bytes, stream, "mxfp4 matmul launch");
}

int mcq4_linear_mxfp4(const void *X, int x_dtype, int64_t ldx, const uint8_t *W, const uint8_t *W_scales, const mcq4_epilogue *e,
                      void *Y, int64_t ldy, int64_t M, int64_t K, int64_t N, void *workspace, size_t workspace_bytes, void *stream) {
    if (!e) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(x_dtype)) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    if (e->activation < 0 || e->activation >= mcq4::MX_ACTS) return fail(MCQ4_ERR_INVALID_ARG, "activation (%d) out of range", e->activation);
    const int es = (int)dt_size(x_dtype);
    if (e->bias) {
        if (e->bias_dtype != x_dtype && e->bias_dtype != MCQ4_DTYPE_F32) return fail(MCQ4_ERR_INVALID_ARG, "bias_dtype must be x_dtype or MCQ4_DTYPE_F32");
        if (!aligned(e->bias, dt_size(e->bias_dtype))) return fail(MCQ4_ERR_ALIGNMENT, "bias must be aligned to its element size");
    }
    if (e->multiply && e->ld_multiply < N) return fail(MCQ4_ERR_SHAPE, "ld_multiply (%lld) < N (%lld)", (long long)e->ld_multiply, (long long)N);
    if (e->residual && e->ld_residual < N) return fail(MCQ4_ERR_SHAPE, "ld_residual (%lld) < N (%lld)", (long long)e->ld_residual, (long long)N);
    if (!aligned(e->multiply, es) || !aligned(e->residual, es))
        return fail(MCQ4_ERR_ALIGNMENT, "multiply and residual must be aligned to their element size");
    auto rows16 = [&](const void *p, int64_t ld) { return !p || (aligned(p, 16) && ld * es % 16 == 0); };
    const mcq4::MxEpilogue epi = {e->bias, e->multiply, e->residual, e->ld_multiply, e->ld_residual, e->bias_dtype, e->activation,
                                  rows16(e->multiply, e->ld_multiply) && rows16(e->residual, e->ld_residual) && aligned(e->bias, 16)};
    return matmul({X, nullptr, x_dtype, ldx, W, W_scales, Y, ldy, M, K, N, &epi}, workspace, workspace_bytes, stream, "mxfp4 linear launch");
}

size_t mcq4_matmul_mxfp4_mxfp4_workspace_bytes(int64_t M, int64_t K, int64_t N) {
    if (M <= 0 || K <= 0 || N <= 0 || K % 32) return 0;
    static const uint8_t any = 0;
    mcq4::MxCall c = {};
    c.Xs = &any; c.M = M; c.K = K; c.N = N;
    return mcq4::mx_workspace_bytes(mcq4::mx_plan(c));
}

int mcq4_matmul_mxfp4_mxfp4(const uint8_t *X, const uint8_t *X_scales, const uint8_t *W, const uint8_t *W_scales, void *Y,
                            int y_dtype, int64_t ldy, int64_t M, int64_t K, int64_t N, void *workspace,
                            size_t workspace_bytes, void *stream) {
    if (!X_scales) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    return matmul({X, X_scales, y_dtype, K / 2, W, W_scales, Y, ldy, M, K, N, nullptr}, workspace, workspace_bytes, stream, "mxfp4 x mxfp4 matmul launch");
}

int mcq4_qk_norm_rope(const mcq4_rope *p, void *stream) {
    if (!p || !p->positions || !p->inv_freq) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(p->dtype)) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    const int64_t es = dt_size(p->dtype);
    if (p->head_dim <= 0 || p->head_dim > 512 || p->head_dim % 8)
        return fail(MCQ4_ERR_SHAPE, "head_dim (%d) must be a multiple of 8 up to 512", p->head_dim);
    if (p->rotary_dim <= 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 8)
        return fail(MCQ4_ERR_SHAPE, "rotary_dim (%d) must be a multiple of 8 up to head_dim (%d)", p->rotary_dim, p->head_dim);
    if (p->T <= 0 || p->T > 1 << 24) return fail(MCQ4_ERR_SHAPE, "T (%lld) out of range", (long long)p->T);
    if (p->axes < 1 || p->axes > mcq4::ROPE_AXES) return fail(MCQ4_ERR_SHAPE, "axes (%d) must be 1 to 4", p->axes);
    if (p->axes > 1 && p->axis_stride < p->T) return fail(MCQ4_ERR_SHAPE, "axis_stride (%lld) < T (%lld)", (long long)p->axis_stride, (long long)p->T);
    if (!aligned(p->positions, 4) || !aligned(p->inv_freq, 16))
        return fail(MCQ4_ERR_ALIGNMENT, "positions must be aligned to 4 bytes, inv_freq to 16");
    mcq4::Rope r = {};
    int64_t sum = 0;
    for (int a = 0; a < mcq4::ROPE_AXES; ++a) {
        if (a < p->axes) {
            if (p->sections[a] < 0) return fail(MCQ4_ERR_SHAPE, "sections must not be negative");
            sum += p->sections[a];
        }
        r.end[a] = (int)std::min<int64_t>(sum, 512);         // axes that are not there begin behind the last pair
    }
    if (2 * sum != p->rotary_dim) return fail(MCQ4_ERR_SHAPE, "sections must add up to rotary_dim / 2 (%d)", p->rotary_dim / 2);
    r.vec = true;
    for (auto [h, o] : {std::pair<const mcq4_rope_heads *, mcq4::RopeHeads *>{&p->q, &r.q}, {&p->k, &r.k}}) {
        if (!h->x || !h->out) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
        if (h->heads <= 0 || h->heads > 65535) return fail(MCQ4_ERR_SHAPE, "heads (%d) out of range", h->heads);
        if (h->token_stride < 0 || h->head_stride < 0 || h->out_token_stride < 0 || h->out_head_stride < 0)
            return fail(MCQ4_ERR_SHAPE, "strides must not be negative");
        if (!aligned(h->x, es) || !aligned(h->out, es)) return fail(MCQ4_ERR_ALIGNMENT, "q, k and their outputs must be aligned to their element size");
        if (h->weight && !valid_dt(h->weight_dtype)) return fail(MCQ4_ERR_INVALID_ARG, "weight_dtype must be MCQ4_DTYPE_F32, F16 or BF16");
        if (h->weight && !aligned(h->weight, dt_size(h->weight_dtype))) return fail(MCQ4_ERR_ALIGNMENT, "a weight must be aligned to its element size");
        r.vec = r.vec && aligned(h->x, 16) && aligned(h->out, 16) &&
                (h->token_stride | h->head_stride | h->out_token_stride | h->out_head_stride) * es % 16 == 0;
        *o = {h->x, h->out, h->weight, h->token_stride, h->head_stride, h->out_token_stride, h->out_head_stride, h->heads, h->weight_dtype, aligned(h->weight, 16)};
    }
    r.positions = p->positions;
    r.inv_freq = p->inv_freq;
    r.axis_stride = p->axis_stride;
    r.T = (int)p->T;
    r.D = p->head_dim;
    r.half = p->rotary_dim / 2;
    r.eps = p->eps;
    r.dt = p->dtype;
    r.pairs = p->interleaved != 0;
    return hip_status(mcq4::launch_qk_rope(r, (hipStream_t)stream), "qk rope launch");
}

int mcq4_kv8_append(const mcq4_kv8_cache *cache, const mcq4_kv8_batch *batch, const void *K, int64_t k_token_stride,
                    int64_t k_head_stride, const void *V, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                    void *stream) {
    mcq4::Kv8Cache c;
    mcq4::Kv8Batch b;
    if (!K || !V) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(dtype)) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    if (int st = check_cache(cache, batch, c, b, true)) return st;
    if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
        return fail(MCQ4_ERR_SHAPE, "strides must not be negative");
    if (!aligned(K, dt_size(dtype)) || !aligned(V, dt_size(dtype))) return fail(MCQ4_ERR_ALIGNMENT, "K and V must be aligned to their element size");
    return hip_status(mcq4::launch_kv8_append(c, b, {K, k_token_stride, k_head_stride}, {V, v_token_stride, v_head_stride}, dtype, (hipStream_t)stream),
                      "kv8 append launch");
}

int mcq4_kv8_read(const mcq4_kv8_cache *cache, const mcq4_kv8_batch *batch, void *K_out, void *V_out, int dtype, void *stream) {
    mcq4::Kv8Cache c;
    mcq4::Kv8Batch b;
    if (!K_out || !V_out) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!valid_dt(dtype)) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F32, F16 or BF16");
    if (int st = check_cache(cache, batch, c, b, false)) return st;
    if (!aligned(K_out, 16) || !aligned(V_out, 16)) return fail(MCQ4_ERR_ALIGNMENT, "K_out and V_out must be 16-byte aligned");
    return hip_status(mcq4::launch_kv8_read(c, b, K_out, V_out, dtype, (hipStream_t)stream), "kv8 read launch");
}

size_t mcq4_kv8_shared_attention_workspace_bytes(const mcq4_kv8_cache *cache, const mcq4_kv8_prefixes *prefix,
                                                 const mcq4_kv8_batch *batch, int32_t heads, int64_t max_prefix, int64_t max_context) {
    mcq4::Kv8Attend a = {};
    mcq4::Kv8Shared x = {};
    if (check_cache(cache, batch, a.cache, a.batch, true) || check_heads(cache, batch, heads, 0, max_context) ||
        check_prefixes(a, batch, prefix, heads, max_prefix, x))
        return 0;
    a.G = heads / cache->kv_heads;
    a.causal = 1;
    a.max_context = (int)std::min<int64_t>(max_context, kMaxDim);
    return shared_bytes(a, x);
}

int mcq4_kv8_shared_attention(const mcq4_kv8_cache *cache, const mcq4_kv8_prefixes *prefix, const mcq4_kv8_batch *batch,
                              const void *q, int64_t q_token_stride, int64_t q_head_stride, int32_t heads, int dtype, void *out,
                              float *lse, float scale, int64_t max_prefix, int64_t max_context, void *workspace,
                              size_t workspace_bytes, void *stream) {
    mcq4::Kv8Attend a = {};
    mcq4::Kv8Shared x = {};
    if (!q || !out) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (dtype != MCQ4_DTYPE_F16 && dtype != MCQ4_DTYPE_BF16) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F16 or BF16");
    if (int st = check_cache(cache, batch, a.cache, a.batch, true)) return st;
    if (int st = check_heads(cache, batch, heads, 0, max_context)) return st;
    if (int st = check_prefixes(a, batch, prefix, heads, max_prefix, x)) return st;
    if (q_token_stride < 0 || q_head_stride < 0) return fail(MCQ4_ERR_SHAPE, "strides must not be negative");
    if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8) return fail(MCQ4_ERR_ALIGNMENT, "rows of q must be 16-byte aligned");
    if (!aligned(out, 16) || !aligned(lse, 4)) return fail(MCQ4_ERR_ALIGNMENT, "out must be 16-byte aligned, lse to 4 bytes");
    a.q = q;
    a.q_token = q_token_stride;
    a.q_head = q_head_stride;
    a.out = out;
    a.lse = lse;
    a.q_dt = dtype;
    a.G = heads / cache->kv_heads;
    a.scale = scale;
    a.causal = 1;
    a.max_context = (int)std::min<int64_t>(max_context, kMaxDim);
    const size_t need = shared_bytes(a, x);
    if (!need) return fail(MCQ4_ERR_SHAPE, "%lld new tokens of %d heads behind %d prefixes are too many", (long long)batch->T, heads, x.S);
    if (!workspace || workspace_bytes < need)
        return fail(MCQ4_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(MCQ4_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    const bool own = mcq4::kv8_shared_own(a, x);
    char *const ws = (char *)workspace + mcq4::COUNTER_BYTES;
    mcq4::kv8_shared_bytes(a, x, &a.pre, ws + (own ? 0 : mcq4::kv8_attend_workspace_bytes(a)));
    hipError_t e = mcq4::launch_kv8_shared(a, x, (hipStream_t)stream);
    if (e == hipSuccess && !own) e = mcq4::launch_kv8_attend(a, ws, (hipStream_t)stream);
    return hip_status(e, "kv8 shared attention launch");
}

int mcq4_kv8_copy_pages(const mcq4_kv8_pool *pool, const int32_t *src, const int32_t *dst, int64_t n, void *stream) {
    mcq4::Kv8Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (!src || !dst) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (n <= 0 || n > kMaxDim) return fail(MCQ4_ERR_SHAPE, "n (%lld) out of range", (long long)n);
    if (!aligned(src, 4) || !aligned(dst, 4)) return fail(MCQ4_ERR_ALIGNMENT, "src and dst must be aligned to 4 bytes");
    if (int st = earlier_status()) return st;
    return hip_status(mcq4::launch_kv8_copy_pages(p, src, dst, n, (hipStream_t)stream), "kv8 copy launch");
}

int mcq4_kv8_fork(const mcq4_kv8_pool *pool, const int32_t *block_table, int64_t table_stride, int64_t batch, int64_t width,
                  const int32_t *lens, const int32_t *parents, int64_t rows, int32_t *out_table, int32_t *out_lens, int32_t release,
                  void *stream) {
    mcq4::Kv8Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (int st = check_table(block_table, table_stride, batch, width, p.page_log)) return st;
    if (!lens || !parents || !out_table || !out_lens) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (rows <= 0 || rows > 1 << 20 || rows * width > kMaxDim) return fail(MCQ4_ERR_SHAPE, "rows (%lld) out of range", (long long)rows);
    if (!aligned(lens, 4) || !aligned(parents, 4) || !aligned(out_table, 4) || !aligned(out_lens, 4))
        return fail(MCQ4_ERR_ALIGNMENT, "lens, parents, out_table and out_lens must be aligned to 4 bytes");
    if (int st = earlier_status()) return st;
    return hip_status(mcq4::launch_kv8_fork(p, {block_table, table_stride, lens, parents, out_table, out_lens, (int)batch, (int)width, (int)rows,
                                                release != 0}, (hipStream_t)stream), "kv8 fork launch");
}

size_t mcq4_kv8_resize_workspace_bytes(const mcq4_kv8_pool *pool, int64_t batch) {
    mcq4::Kv8Pool p;
    if (check_pool(pool, p) || batch <= 0 || batch > 1 << 20) return 0;
    return mcq4::COUNTER_BYTES + mcq4::kv8_resize_bytes(p, batch);
}

int mcq4_kv8_resize(const mcq4_kv8_pool *pool, int32_t *block_table, int64_t table_stride, int64_t batch, int64_t width,
                    const int32_t *lens, const int32_t *new_lens, int32_t *missing, void *workspace, size_t workspace_bytes, void *stream) {
    mcq4::Kv8Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (int st = check_table(block_table, table_stride, batch, width, p.page_log)) return st;
    if (!lens || !new_lens || !missing) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!aligned(lens, 4) || !aligned(new_lens, 4) || !aligned(missing, 4))
        return fail(MCQ4_ERR_ALIGNMENT, "lens, new_lens and missing must be aligned to 4 bytes");
    const size_t need = mcq4::COUNTER_BYTES + mcq4::kv8_resize_bytes(p, batch);
    if (!workspace || workspace_bytes < need)
        return fail(MCQ4_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(MCQ4_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    if (int st = earlier_status()) return st;
    return hip_status(mcq4::launch_kv8_resize(p, {block_table, table_stride, lens, new_lens, missing, (int)batch, (int)width},
                                              (char *)workspace + mcq4::COUNTER_BYTES, (hipStream_t)stream), "kv8 resize launch");
}

size_t mcq4_kv8_compact_workspace_bytes(const mcq4_kv8_pool *pool) {
    mcq4::Kv8Pool p;
    return check_pool(pool, p) ? 0 : mcq4::COUNTER_BYTES + mcq4::kv8_compact_bytes(p);
}

int mcq4_kv8_compact(const mcq4_kv8_pool *pool, int32_t *names, int32_t *live, void *workspace, size_t workspace_bytes, void *stream) {
    mcq4::Kv8Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (!names || !live) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (!aligned(names, 4) || !aligned(live, 4)) return fail(MCQ4_ERR_ALIGNMENT, "names and live must be aligned to 4 bytes");
    const size_t need = mcq4::COUNTER_BYTES + mcq4::kv8_compact_bytes(p);
    if (!workspace || workspace_bytes < need)
        return fail(MCQ4_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16)) return fail(MCQ4_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    if (int st = earlier_status()) return st;
    return hip_status(mcq4::launch_kv8_compact(p, names, live, (char *)workspace + mcq4::COUNTER_BYTES, (hipStream_t)stream), "kv8 compact launch");
}

int mcq4_kv8_rename(int32_t *block_table, int64_t table_stride, int64_t batch, int64_t width, const int32_t *names, int64_t num_pages, void *stream) {
    if (int st = check_table(block_table, table_stride, batch, width, 4)) return st;
    if (!names) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (num_pages <= 0 || num_pages > kMaxDim) return fail(MCQ4_ERR_SHAPE, "num_pages (%lld) out of range", (long long)num_pages);
    if (!aligned(names, 4)) return fail(MCQ4_ERR_ALIGNMENT, "names must be aligned to 4 bytes");
    if (int st = earlier_status()) return st;
    return hip_status(mcq4::launch_kv8_rename(block_table, table_stride, batch, (int)width, names, num_pages, (hipStream_t)stream), "kv8 rename launch");
}

size_t mcq4_kv8_attention_workspace_bytes(const mcq4_kv8_cache *cache, const mcq4_kv8_batch *batch, int32_t heads,
                                          int32_t causal, int32_t window, int64_t max_context) {
    mcq4::Kv8Attend a = {};
    if (check_cache(cache, batch, a.cache, a.batch, true) || check_heads(cache, batch, heads, window, max_context)) return 0;
    a.G = heads / cache->kv_heads;
    a.causal = causal != 0;
    a.window = window;
    a.max_context = (int)std::min<int64_t>(max_context, kMaxDim);
    const size_t n = mcq4::kv8_attend_workspace_bytes(a);
    return n ? n + mcq4::COUNTER_BYTES : 0;
}

int mcq4_kv8_attention(const mcq4_kv8_cache *cache, const mcq4_kv8_batch *batch, const void *q, int64_t q_token_stride,
                       int64_t q_head_stride, int32_t heads, int dtype, void *out, float *lse, float scale, int32_t causal,
                       int32_t window, int64_t max_context, void *workspace, size_t workspace_bytes, void *stream) {
    mcq4::Kv8Attend a = {};
    if (!q || !out) return fail(MCQ4_ERR_INVALID_ARG, "null pointer");
    if (dtype != MCQ4_DTYPE_F16 && dtype != MCQ4_DTYPE_BF16) return fail(MCQ4_ERR_INVALID_ARG, "dtype must be MCQ4_DTYPE_F16 or BF16");
    if (int st = check_cache(cache, batch, a.cache, a.batch, true)) return st;
    if (int st = check_heads(cache, batch, heads, window, max_context)) return st;
    if (q_token_stride < 0 || q_head_stride < 0) return fail(MCQ4_ERR_SHAPE, "strides must not be negative");
    if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8) return fail(MCQ4_ERR_ALIGNMENT, "rows of q must be 16-byte aligned");
    if (!aligned(out, 16) || !aligned(lse, 4)) return fail(MCQ4_ERR_ALIGNMENT, "out must be 16-byte aligned, lse to 4 bytes");
    a.q = q;
    a.q_token = q_token_stride;
    a.q_head = q_head_stride;
    a.out = out;
    a.lse = lse;
    a.q_dt = dtype;
    a.G = heads / cache->kv_heads;
    a.scale = scale;
    a.causal = causal != 0;
    a.window = window;
    a.max_context = (int)std::min<int64_t>(max_context, kMaxDim);
    const size_t n = mcq4::kv8_attend_workspace_bytes(a), need = n ? n + mcq4::COUNTER_BYTES : 0;
    if (need && (!workspace || workspace_bytes < need))
        return fail(MCQ4_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (need && !aligned(workspace, 16)) return fail(MCQ4_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    return hip_status(mcq4::launch_kv8_attend(a, need ? (char *)workspace + mcq4::COUNTER_BYTES : nullptr, (hipStream_t)stream),
                      "kv8 attention launch");
}

}  // extern "C"
