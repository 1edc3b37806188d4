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

// Output columns of such a launch's tiles, CUs of an XCD, and workgroups: a split last
// round has up to as many as the GPU has CUs.
constexpr int moe_tile_columns(int tile_rows, bool gated) { return (tile_rows == 256 ? 256 : 128) / (gated ? 2 : 1); }
inline int moe_xcd_cus(int cus) { return cus >= 8 ? cus / 8 : 1; }
inline int64_t moe_product_grid(const MoePlan& plan, int n, bool gated, int xcd_cus) {
    const int columns = moe_tile_columns(plan.tile_rows, gated);
    const int64_t tiles = static_cast<int64_t>(plan.max_tiles) * ((n + columns - 1) / columns);
    return (tiles + 7) / 8 * 8 + 8 + (plan.tile_rows == 256 ? 8 * static_cast<int64_t>(xcd_cus) : 0);
}

constexpr int kMoeManyTiles = 64;

// What of a launch's (row tile, column tile) pairs an XCD's workgroups take; workgroup b
// runs on XCD b % 8, which walks its share in groups of 4 row tiles: they share W in its
// L2 where they are one expert's, and their A over the columns. With many row tiles a share is a
// contiguous range; with few, in which a range's full and partly filled tiles
// would not even out, an eighth of the columns of every row tile (and a range of
// the columns that are left over). us a call by an eighth and by ranges, top 2 of 8 experts of 4096 x
// 14336: 13 row tiles 356 and 387, 12 623 and 613, 19 985 and 992, 52 2531 and 2602, 67 3288
// and 3375, 101 4860 and 5040; 24 of 2000 x 1000: 24 tiles 43.8 and 42.4; 64 of 2048 x 1024: 154 431
// and 432, 292 819 and 846; 8 of 2048 x 1024: 517 1630 and 1611; 256 of 4096 x 2048: 256 1938 and
// 1829. Beyond the limit neither is the better one throughout. Where tiles split, what an XCD's CUs would run in a
// last round that is at most half full runs in two parts (halves of the columns), at
// most a quarter full in four (of the rows, too: parts 0 and 1 the upper, 2 and 3 the lower).
struct MoeShare {
    int tiles_m, tiles_n, xcd, eighth, own, per, rem, mine, rest, parts;
};
__host__ __device__ __forceinline__ MoeShare moe_share(int xcd, int tiles_m, int tiles_n, int xcd_cus, bool splits) {
    const int eighth = tiles_m < kMoeManyTiles ? tiles_n >> 3 : 0;  // columns of each XCD's own
    const int own = eighth * tiles_m, shared = (tiles_n - 8 * eighth) * tiles_m;
    const int per = shared >> 3, rem = shared & 7;
    const int mine = own + per + (xcd < rem), rest = splits ? mine % xcd_cus : 0;
    const int parts = 2 * rest > xcd_cus || rest == 0 ? 1 : 4 * rest > xcd_cus ? 2 : 4;
    return {tiles_m, tiles_n, xcd, eighth, own, per, rem, mine, rest, parts};
}
// The XCD's i-th workgroup's: which of its pairs (none from `mine` on), and which part of it.
__host__ __device__ __forceinline__ void moe_part(const MoeShare& s, int& i, int& part) {
    const int whole = s.mine - s.rest, j = i - whole;
    part = i < whole ? 0 : j % s.parts;
    i = i < whole ? i : whole + j / s.parts;
}
__host__ __device__ __forceinline__ bool moe_splits(const MoeShare& s, int i) { return s.parts > 1 && i >= s.mine - s.rest; }
__host__ __device__ __forceinline__ void moe_pair(const MoeShare& s, int i, int& row, int& column) {
    constexpr int GM = 4;
    const bool is_own = i < s.own;
    const int wide = is_own ? s.eighth : s.tiles_n - 8 * s.eighth;
    const int t = is_own ? i : s.xcd * s.per + min(s.xcd, s.rem) + i - s.own;
    const int group = t / (GM * wide), first_m = group * GM;
    const int gsize = min(s.tiles_m - first_m, GM);
    row = first_m + (t % (GM * wide)) % gsize;
    column = (t % (GM * wide)) / gsize + (is_own ? s.xcd * s.eighth : 8 * s.eighth);
}

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

// f32(g * u / (1 + exp(-g))) with what is inside in 64 bits, to 2^-50 of the value, so
// that about one value in 2^25 is rounded to the neighbour of the nearest f32:
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
