// Which kernel an MXFP4 product takes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdlib.h>

#include "mx_gemm.h"

namespace mcq4 {

namespace {

struct Tile { int m, n; };
Tile tile_of(int kind) {
    switch (kind) {
        case MX_256x256: return {256, 256};
        case MX_128x256: return {128, 256};
        case MX_128x128: return {128, 128};
        case MX_MID_64x64: return {64, 64};
        case MX_MID_32x64: return {32, 64};
        case MX_MID_32x32: return {32, 32};
        default: return {64, 128};
    }
}

// The copies of the LDS kernels count bytes in 31 bits from a tile's first row.
bool fits(const MxCall &c) {
    const int64_t most = (int64_t)1 << 31;
    if (256 * (c.K / 2) >= most) return false;
    if (c.Xs) return true;
    return 256 * std::max<int64_t>(c.x_dt == DT_F32 ? 3 * (c.K + 128) : 0, c.ldx) * 2 < most;
}

}  // namespace

MxPlan mx_plan(const MxCall &c) {
    MxPlan p = {MX_DIRECT, 1, 0};
    const bool f32 = !c.Xs && c.x_dt == DT_F32;
    const int64_t steps = c.Xs ? (c.K + 127) / 128 : (c.K + 127) / 128 * (f32 ? 3 : 1);     // 128 elements of K each
    if (fits(c)) {
        if (c.M > 64) p.kind = c.Xs ? MX_128x128 : MX_64x128;
        auto tiles = [&](int kind) { const Tile t = tile_of(kind); return ((c.M + t.m - 1) / t.m) * ((c.N + t.n - 1) / t.n); };
        if (c.M > 64 && tiles(MX_256x256) >= 128) p.kind = MX_256x256;
        else if (c.M > 64 && !c.Xs && tiles(MX_128x256) >= 128) p.kind = MX_128x256;
        if (const char *v = opt("MCQ4_MX_PATH")) p.kind = std::max(0, std::min(MX_KINDS - 1, atoi(v)));
        if (c.Xs && (p.kind == MX_128x256 || p.kind == MX_64x128)) p.kind = MX_128x128;
        if (c.Xs && p.kind == MX_MID_64x128) p.kind = MX_MID_64x64;
        if (c.Xs && p.kind == MX_MID_32x64) p.kind = MX_MID_32x32;
        if (p.kind != MX_DIRECT) {
            const int64_t t = tiles(p.kind), want = p.kind >= MX_128x128 ? 512 : 256;
            while (t * p.S * 2 <= want && steps / (p.S * 2) >= 4 && p.S < 16) p.S *= 2;
            if (const char *v = opt("MCQ4_MX_SPLIT")) p.S = std::max(1, std::min(16, atoi(v)));
            p.S = (int)std::min<int64_t>(p.S, steps);
            if (p.kind >= MX_MID_64x128 && t > COUNTER_SLOTS) p.S = 1;
        }
    }
    if (p.kind != MX_DIRECT) {
        if (f32) p.bytes += 2 * (size_t)mx_pieces(c.M, c.K);
        if (p.S > 1) {
            const Tile t = tile_of(p.kind);
            const int64_t tm = (c.M + t.m - 1) / t.m, tn = (c.N + t.n - 1) / t.n;
            p.bytes += p.kind >= MX_MID_64x128 ? (size_t)p.S * tm * t.m * tn * t.n * sizeof(float) : (size_t)p.S * c.M * mx_ldp(c.N) * sizeof(float);
        }
    }
    return p;
}

size_t mx_workspace_bytes(const MxCall &c) {
    const size_t n = mx_plan(c).bytes;
    return n ? n + COUNTER_BYTES : 0;
}

hipError_t launch_mx(const MxCall &c, void *scratch, hipStream_t s) {
    const MxPlan p = mx_plan(c);
    if (p.kind == MX_DIRECT) return launch_mx_direct(c, s);
    if (p.kind >= MX_MID_64x128) return launch_mx_mid(c, p, scratch, s);
    return c.Xs ? launch_mx_gemm4(c, p, scratch, s) : launch_mx_gemm(c, p, scratch, s);
}

}  // namespace mcq4
