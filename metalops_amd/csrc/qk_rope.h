// Norms of queries' and keys' heads and their rotation by positions (qk_rope.hip).
#pragma once

#include "mx_common.h"

namespace mcq4 {

constexpr int ROPE_AXES = 4;
struct RopeHeads {                 // [T][heads][D], channels neighbours; strides in elements
    const void *x;
    void *y;
    const void *weight;            // [D] or null
    int64_t token, head, y_token, y_head;
    int heads, weight_dt;
    bool weight_vec;               // at a 16-byte aligned address
};
struct Rope {
    RopeHeads q, k;
    const int32_t *positions;      // [axes][axis_stride]
    const float *inv_freq;         // [half]
    int64_t axis_stride;
    int T, D, half;                // pairs that are rotated
    int end[ROPE_AXES];            // axis a turns pairs end[a - 1] .. end[a] - 1
    float eps;
    int dt, pairs;                 // pairs: a pair is channels 2 i and 2 i + 1, else i and i + half
    bool vec;                      // all rows at 16-byte aligned addresses
};
hipError_t launch_qk_rope(const Rope &r, hipStream_t s);

}  // namespace mcq4
