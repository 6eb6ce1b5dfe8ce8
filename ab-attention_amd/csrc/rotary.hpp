// One call of the rotary kernel.
#pragma once

#include "window.hpp"

namespace ab {

constexpr int kMaxAxes = 4;

struct RotaryCall {
    const void* in[2];   // Q and K (heads[1] = 0: none)
    void* out[2];
    Rows in_rows[2], out_rows[2];
    const void* positions;  // [tokens][axes], or [batch][tokens][axes] with per_batch
    double step[kMaxAxes];  // log2(theta) * 2 / dims of the axis (joint: step[0], of all dims)
    double ratio[kMaxAxes];  // 2^-step: from a pair's frequency to the next one's
    int32_t pairs[kMaxAxes];
    int32_t axes, heads[2];
    int32_t position_kind;  // 0 int32, 1 int64, 2 float32
    int32_t turned;         // dims of all axes
    uint32_t total, tokens, units;
    int32_t heads_each;
    float sign;             // 1, or -1 for the gradient
    int32_t per_batch, joint;  // 0 or 1
};

int launch_rotary(const RotaryCall& call, int dtype, bool halves, hipStream_t stream);

}  // namespace ab
