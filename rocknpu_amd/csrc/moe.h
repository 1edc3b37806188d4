// What the kernels of an expert feed-forward share: the plan, which the routing
// writes and the products read (include/rocknpu_moe.h).
#pragma once

#include "common.h"
#include "rocknpu_moe.h"

#include <algorithm>

namespace rk {

// A plan's parts, all int32. `tiles` lists the products' row tiles, two words
// each: the expert and the tile's first row in `order`; a tile ends after tile_rows
// rows or with its expert's. `place` is where each choice stands in `order` (-1:
// nothing was chosen). `counts` is the routing's own: each block's choices by expert.
struct MoePlan {
    int32_t* tile_count;  // [1], the first of the header's words
    int32_t* offsets;     // [experts + 1]
    int32_t* order;       // [rows]
    int32_t* place;       // [rows]
    int32_t* tiles;       // [max_tiles][2]
    int32_t* counts;      // [blocks][experts]
    int rows, experts, top_k;
    int tile_rows, max_tiles;
    int block, blocks;  // choices of a counting block, and blocks
};

constexpr int kMoeHeader = 16;
constexpr int kMoeCountThreads = 1024;

// Rows of a product's tile: 256 x 256 tiles where an expert has rows for them, 64 x
// 128, which stream weights with two workgroups a CU, where it has few. us a call by 64
// and by 256 at a mean of 64, 80, 96 and 128 rows an expert: 64 experts of 2048 x 1024
// 141 and 145, 159 and 162, 173 and 169, 199 and 183; 128 of 2048 x 768 214 and 215, 233
// and 229, 255 and 246, 306 and 274; 8 of 4096 x 14336 408 and 393, 412 and 407, 439 and
// 424, 515 and 449; 16 of 2048 x 1024 46 and 49, 48 and 52, 49 and 53, 74 and 67.
inline int moe_tile_rows(int64_t rows, int experts) {
    return rows >= static_cast<int64_t>(96) * experts ? 256 : 64;
}

// The plan of such a call at `base` (which may be null), and its words.
inline MoePlan moe_plan(int64_t tokens, int experts, int top_k, int32_t* base, size_t* words) {
    MoePlan p{};
    p.rows = static_cast<int>(tokens * top_k);
    p.experts = experts;
    p.top_k = top_k;
    p.tile_rows = moe_tile_rows(p.rows, experts);
    p.max_tiles = p.rows / p.tile_rows + (p.rows < experts ? p.rows : experts);
    // 64 tokens a counting block, more where that would be over 256 blocks
    const int64_t per_block = 64 * std::max<int64_t>((tokens + 64 * 256 - 1) / (64 * 256), 1);
    p.block = static_cast<int>(per_block * top_k);
    p.blocks = static_cast<int>((tokens + per_block - 1) / per_block);
    size_t at = 0;
    const auto take = [&](size_t n) {
        int32_t* q = base ? base + at : nullptr;
        at += n;
        return q;
    };
    p.tile_count = take(kMoeHeader);
    p.offsets = take(static_cast<size_t>(experts) + 1);
    p.order = take(p.rows);
    p.place = take(p.rows);
    p.tiles = take(static_cast<size_t>(p.max_tiles) * 2);
    p.counts = take(p.blocks > 1 ? static_cast<size_t>(p.blocks) * experts : 0);
    if (words) *words = at;
    return p;
}

// Whether a plan of that size is one that the kernels can take. moe_route.hip.
bool moe_size_ok(int64_t tokens, int32_t experts, int32_t top_k);

}  // namespace rk
