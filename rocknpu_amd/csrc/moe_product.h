// The experts' products: over a plan's tiles (moe_product.hip), or for a few tokens
// choice by choice (moe_decode.hip).
#pragma once

#include "moe.h"

namespace rk {

// Rows of `a` [.., k] (of the token of each choice where gated, else of the choice's
// place in the plan's order) times w[0] (and w[1]) [experts][n][k], into out
// [rows][ldo] in the plan's order, zeros behind n; ldo is at most n's next
// multiple of 64.
struct MoeProduct {
    const int8_t* a;
    const float* a_scales;
    const int8_t* w[2];
    const float* w_scales[2];
    float* out;
    int n, k, ldo, top_k;
    int xcd_cus;  // CUs of an XCD, filled in by the launch
};
int launch_moe_product(MoeProduct p, bool gated, const MoePlan& plan, hipStream_t stream);


// The whole feed-forward of a few tokens, by their ids. `values` holds SwiGLU's rows
// [tokens * top_k][ffn_pad].
struct MoeDecode {
    const int8_t* a;
    const float* a_scales;
    const int8_t* gate;
    const int8_t* up;
    const int8_t* down;
    const float* gate_scales;
    const float* up_scales;
    const float* down_scales;
    const int32_t* ids;
    const float* weights;
    float* values;
    int tokens, experts, top_k, hidden, hidden_pad, ffn, ffn_pad;
};
bool moe_decodes(int64_t tokens, int experts, int top_k, int ffn_pad);
int launch_moe_decode(const MoeDecode& p, uint32_t out_type, void* out, int64_t out_row, hipStream_t stream);

// f32(g * u / (1 + exp(-g))) with what is inside in 64 bits, to 2^-50 of the value:
// exp(-g) = 2^n 2^r with n = rint(-g log2(e)), |r| <= 1/2 in two parts of log2(e),
// 2^r by the polynomial through its values at the 11 Chebyshev nodes of [-1/2, 1/2]
// (off by 2^-51.5 at most), the division by the reciprocal's Newton step and one
// of the quotient. In the exponential g is held to +-693, where the value is that of
// 1 + exp(-g) = 1, or 0 in f32.
__device__ __forceinline__ float swiglu(float gate, float up) {
    const double x = static_cast<double>(gate) * static_cast<double>(up);
    const double g = static_cast<double>(__builtin_amdgcn_fmed3f(gate, -693.0f, 693.0f));
    const double n = rint(g * -0x1.71547652b82fep+0);
    double r = fma(g, -0x1.71547652b82fep+0, -n);
    r = fma(g, -0x1.777d0ffda0d24p-56, r);
    double p = 0x1.e6063f7217bc6p-28;
    p = fma(p, r, 0x1.b675bca4eeebbp-24);
    p = fma(p, r, 0x1.62bfd47773353p-20);
    p = fma(p, r, 0x1.ffcb54062e698p-17);
    p = fma(p, r, 0x1.430913096fd9fp-13);
    p = fma(p, r, 0x1.5d87fe9d7a584p-10);
    p = fma(p, r, 0x1.3b2ab6fba1ddap-7);
    p = fma(p, r, 0x1.c6b08d703ce49p-5);
    p = fma(p, r, 0x1.ebfbdff82c598p-3);
    p = fma(p, r, 0x1.62e42fefa3a19p-1);
    p = fma(p, r, 1.0);
    const double d = 1.0 + ldexp(p, static_cast<int>(n));
    double y = __builtin_amdgcn_rcp(d);
    y = fma(fma(-d, y, 1.0), y, y);
    const double q = x * y;
    return static_cast<float>(fma(fma(-d, q, x), y, q));
}

}  // namespace rk
