// Which kernel an MXFP4 product takes, and over how many workgroups it splits K.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdlib.h>

#include "mx_gemm.h"

namespace mcq4 {

namespace {

struct Tile { int m, n, waves; };      // logarithms; waves that divide K
constexpr Tile TILE[MX_KINDS] = {{4, 4, 0}, {8, 8, 0}, {7, 8, 0}, {7, 7, 0}, {6, 7, 0}, {6, 6, 2}, {5, 6, 3}, {5, 5, 3}};

// What a call takes, in microseconds, as measured over M = 1 .. 2048, K = 512 .. 14336 and
// N = 512 .. 14336 with every kernel and 1, 2, 4 and 8 splits (5600 timings in HIP graphs, weights
// from memory) and fitted kernel by kernel; 5 to 12% off a timing.  Over those sizes the
// choice by it is 1 to 2.5% slower than the fastest one on average, and 29% at most.
//   step      a step is 128 elements of K of a wave's tile; taken by every round of 256 workgroups,
//   share     and by the workgroups' number over 256,
//   round     a round's start and end,
//   join ..   with more than one split: once, for each split (of a million results where
//             mx_sum_kernel adds them), and for workgroups / 256.
struct Cost { float fixed, step, share, round, join, join_split, join_wgs; };
constexpr Cost NEVER = {1e30f, 0, 0, 0, 0, 0, 0};
constexpr Cost COST_16[MX_KINDS] = {        // 16-bit X
    {}, {3.53f, 1.89f, 0.91f, 5.13f, 5.25f, 1.13f, 0}, {3.47f, 1.14f, 0.55f, 1.92f, 4.25f, 1.28f, 0}, {3.63f, 0.81f, 0.22f, 0, 4.02f, 1.35f, 0},
    {3.13f, 0.55f, 0.14f, 0, 3.37f, 1.67f, 0}, {2.37f, 0.91f, 0.56f, 2.40f, 0.82f, 1.12f, 0.85f}, {2.58f, 1.35f, 0.76f, 1.69f, 1.16f, 0.45f, 0.97f},
    {2.24f, 0.74f, 0.53f, 1.80f, 1.14f, 0.35f, 0.51f}};
constexpr Cost COST_F32[MX_KINDS] = {       // fp32 X, its conversion included
    {}, {7.45f, 2.12f, 0.71f, 7.35f, 1.23f, 1.21f, 0}, {9.83f, 1.27f, 0.56f, 0, 1.72f, 1.18f, 0}, {7.53f, 1.02f, 0.19f, 0, 2.91f, 1.00f, 0},
    {5.78f, 0.84f, 0, 0, 2.60f, 1.43f, 0}, {5.07f, 0.92f, 0.66f, 1.87f, 0.48f, 1.19f, 0.37f}, {5.67f, 1.30f, 0.99f, 1.05f, 0.44f, 0.50f, 0.92f},
    {5.18f, 0.72f, 0.65f, 1.53f, 0.51f, 0.36f, 0.44f}};
constexpr Cost COST_4[MX_KINDS] = {         // microscaled X
    {}, {3.63f, 0.64f, 0.39f, 3.94f, 5.35f, 1.12f, 0}, NEVER, {4.09f, 0.29f, 0.14f, 0, 3.30f, 1.62f, 0},
    NEVER, {2.16f, 0.39f, 0.34f, 2.58f, 0.94f, 1.07f, 0.84f}, NEVER, {2.28f, 0.44f, 0.22f, 1.82f, 1.05f, 0.34f, 0.64f}};
// The direct kernel: for each batch of steps whose loads go out together, by the workgroups' steps, by them
// and M, and by rounds.  Up to 8 rows (fp32 X: 128), beyond which it never was the fastest.
struct DirectCost { float fixed, batch, step, step_m, round; int most_m; };
constexpr DirectCost DIRECT_16 = {0, 4.58f, 0.062f, 0.0073f, 0.07f, 8}, DIRECT_4 = {0, 4.24f, 0.037f, 0.0045f, 0.30f, 8},
                     DIRECT_F32 = {0.76f, 1.97f, 0.057f, 0, 0.24f, 128};

int64_t ceil_shift(int64_t a, int b) { return (a + ((int64_t)1 << b) - 1) >> b; }

// The copies of the LDS kernels count bytes in 31 bits from a tile's first row.
bool fits(const MxCall &c) {
    const int64_t most = (int64_t)1 << 31;
    if (256 * (c.K / 2) >= most) return false;
    if (c.Xs) return true;
    return 256 * std::max<int64_t>(c.x_dt == DT_F32 ? 3 * (c.K + 128) : 0, c.ldx) * 2 < most;
}

}  // namespace

// Asked for twice a call, so in shifts and products: about 0.2 us.
MxPlan mx_plan(const MxCall &c) {
    MxPlan p = {MX_DIRECT, 1, 0};
    const bool f32 = !c.Xs && c.x_dt == DT_F32;
    const int64_t steps1 = ceil_shift(c.K, 7), steps = steps1 * (f32 ? 3 : 1);
    auto tiles = [&](int kind) { return ceil_shift(c.M, TILE[kind].m) * ceil_shift(c.N, TILE[kind].n); };
    if (fits(c)) {
        const DirectCost &d = c.Xs ? DIRECT_4 : f32 ? DIRECT_F32 : DIRECT_16;
        const Cost *costs = c.Xs ? COST_4 : f32 ? COST_F32 : COST_16;
        float best = 1e30f;
        if (c.M <= d.most_m) {
            const int64_t t = tiles(MX_DIRECT);
            const int at_once = mx_direct_waves(c.K) * mx_direct_batch(c);
            best = d.fixed + d.batch * (float)((steps1 + at_once - 1) / at_once) + (float)(t * steps) / 256 * (d.step + d.step_m * (float)c.M) + d.round * (float)ceil_shift(t, 8);
        }
        const float results = (float)c.M * (float)c.N * 1e-6f;
        for (int kind = 1; kind < MX_KINDS; ++kind) {
            const Cost &k = costs[kind];
            if (k.fixed >= best) continue;
            const int64_t t = tiles(kind);
            const bool mid = kind >= MX_MID_64x64;
            for (int log = 0; log <= 3; ++log) {
                // A split has two steps at least and makes no more than 1023 workgroups; tiles have tickets.
                if (log && ((steps1 >> log) < 2 || (t << log) >= 1024 || (mid && t > COUNTER_SLOTS))) break;
                const float w = (float)(t << log) / 256, rounds = (float)ceil_shift(t << log, 8), per = (float)steps / (float)(1 << (log + TILE[kind].waves));
                float cost = k.fixed + per * (k.step * rounds + k.share * w) + k.round * rounds;
                if (log) cost += k.join + k.join_split * (float)(1 << log) * (mid ? 1.f : results) + k.join_wgs * w;
                if (cost < best) { best = cost; p.kind = kind; p.S = 1 << log; }
            }
        }
        if (const char *v = opt("MCQ4_MX_PATH")) {
            p.kind = std::max(0, std::min((int)MX_KINDS - 1, atoi(v)));
            if (c.Xs && (p.kind == MX_128x256 || p.kind == MX_64x128)) p.kind = MX_128x128;
            if (c.Xs && p.kind == MX_MID_32x64) p.kind = MX_MID_32x32;
            p.S = 1;
        }
        if (const char *v = opt("MCQ4_MX_SPLIT"))
            if (p.kind != MX_DIRECT && (p.kind < MX_MID_64x64 || tiles(p.kind) <= COUNTER_SLOTS)) p.S = (int)std::min<int64_t>(std::max(1, std::min(16, atoi(v))), steps);
    }
    if (p.kind != MX_DIRECT) {
        if (f32) p.bytes += 2 * (size_t)mx_pieces(c.M, c.K);
        if (p.S > 1) {
            const size_t tile = (size_t)1 << (TILE[p.kind].m + TILE[p.kind].n);
            p.bytes += p.kind >= MX_MID_64x64 ? (size_t)p.S * tiles(p.kind) * tile * sizeof(float) : (size_t)p.S * c.M * mx_ldp(c.N) * sizeof(float);
        }
    }
    return p;
}

size_t mx_workspace_bytes(const MxPlan &p) { return p.bytes ? p.bytes + COUNTER_BYTES : 0; }

hipError_t launch_mx(const MxCall &c, const MxPlan &p, void *scratch, hipStream_t s) {
    if (p.kind == MX_DIRECT) return launch_mx_direct(c, s);
    if (p.kind >= MX_MID_64x64) return launch_mx_mid(c, p, scratch, s);
    return c.Xs ? launch_mx_gemm4(c, p, scratch, s) : launch_mx_gemm(c, p, scratch, s);
}

}  // namespace mcq4
