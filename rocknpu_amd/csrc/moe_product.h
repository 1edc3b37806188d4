// The experts' products over a plan's tiles. moe_product.hip.
#pragma once

#include "moe.h"

namespace rk {

// Rows of `a` [.., k] (of the token of each choice where gated, else of the choice's
// place in the plan's order) times w[0] (and w[1]) [experts][n][k], into out
// [rows][n] in the plan's order.
struct MoeProduct {
    const int8_t* a;
    const float* a_scales;
    const int8_t* w[2];
    const float* w_scales[2];
    float* out;
    int n, k, top_k;
    int xcd_cus;  // CUs of an XCD, filled in by the launch
};
int launch_moe_product(MoeProduct p, bool gated, const MoePlan& plan, hipStream_t stream);

}  // namespace rk
