// xm_gate.cuh -- the gate of the gated linear recurrence.
#pragma once

#include "xm_common.cuh"

namespace xm {

// keep = sigmoid(f), take = sigmoid(-f) = 1 - keep, each with its own relative
// precision: with t = exp(-|f|) <= 1 the larger is r = 1 / (1 + t) and the smaller
// t r, so no difference of nearby values is formed and nothing overflows.
struct Gate {
    float keep, take;
};
__device__ __forceinline__ Gate gate_of(float f) {
    const float t = ex2_approx(-fabsf(f) * kLog2e);
    const float r = rcp_approx(1.0f + t), s = t * r;
    return f >= 0.0f ? Gate{r, s} : Gate{s, r};
}

}  // namespace xm
