/*
 * rocknpu_moe.h — a feed-forward made of experts, on device buffers: which
 * experts a token goes to, and the experts' W8A8 products.
 *
 * No counterpart in the reference, whose plugin takes plain MUL_MAT nodes only
 * (adapters/ggml-rocknpu/src/ggml-rocknpu.cpp:614-715); the products' arithmetic
 * is that of its W8A8 route (crates/rocknpu-capi/src/lib.rs:614-709), as in
 * rocknpu_hip_quantize_a8 and rocknpu_hip_gemm_w8a8.
 *
 * Every pointer inside the structures is a DEVICE pointer, the structures
 * themselves are host memory read during the call; `stream` is a hipStream_t.
 * Calls validate what the host can see, enqueue and return without
 * synchronising or allocating. Status codes are those of rocknpu.h (0 ok, -1
 * invalid argument, -3 launch failure). Types are ROCKNPU_TYPE_* of
 * rocknpu_hip.h.
 */
#ifndef ROCKNPU_MOE_H
#define ROCKNPU_MOE_H

#include <stddef.h>
#include <stdint.h>

#include "rocknpu_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ROCKNPU_MOE_SOFTMAX 0
#define ROCKNPU_MOE_SIGMOID 1
#define ROCKNPU_MOE_MAX_EXPERTS 1024
#define ROCKNPU_MOE_MAX_TOP_K 64
#define ROCKNPU_MOE_MAX_GROUPS 64
#define ROCKNPU_MOE_MAX_ROWS (1 << 28) /* tokens * top_k */

typedef struct rocknpu_moe_route_args {
    const void * logits; /* [tokens][experts] of `type`, rows logits_row elements apart */
    const float * bias;  /* [experts], added to the scores for the choice only, or NULL */
    int32_t * ids;       /* [tokens][top_k] */
    float * weights;     /* [tokens][top_k] */
    int32_t * plan;      /* rocknpu_hip_moe_plan_words words: the rows in order of expert, for rocknpu_hip_moe_experts */
    int64_t tokens, logits_row;
    uint32_t type;
    int32_t experts, top_k;
    int32_t groups;      /* of experts / groups neighbours each; 1: none */
    int32_t top_groups;  /* groups that a token may choose from; their experts are at least top_k */
    int32_t group_top;   /* a group's rank: 1, its best expert's rank; 2, the sum of its two best scores + bias */
    int32_t score;       /* ROCKNPU_MOE_SOFTMAX over the token's logits, or ROCKNPU_MOE_SIGMOID of each */
    int32_t normalise;   /* weights are divided by their sum + 1e-20 */
    float factor;        /* and multiplied by this */
} rocknpu_moe_route_args;

/* Chooses top_k experts for every token. Experts are ranked by score + bias in 64
 * bits, without a bias by the logits themselves, equal ones by index; a logit of
 * -inf, or a bias of -inf or NaN, is an expert that cannot be chosen. With groups
 * only the experts of the top_groups groups of highest rank can (equal groups by
 * index; a group without group_top experts that can be chosen ranks lowest). ids
 * are in order of rank; weights are the chosen scores (without bias), normalised and multiplied. Where
 * less than top_k experts can be chosen the last ids are -1 and their weights 0.
 * A row that holds a NaN or +inf has its lowest experts and NaN weights. Outputs
 * overlap neither each other nor what is read.
 *
 * The plan begins with 16 words of its own, then offsets [experts + 1] and order
 * [tokens * top_k]: order[offsets[e]] .. order[offsets[e + 1] - 1] are, ascending,
 * the numbers token * top_k + place of the choices that fell on expert e, and what
 * follows offsets[experts] is -1. The rest is the library's. */
int rocknpu_hip_moe_route(const rocknpu_moe_route_args * args, void * stream);

/* Words of such a plan. Host code only. */
int rocknpu_hip_moe_plan_words(int64_t tokens, int32_t experts, int32_t top_k, size_t * words);

typedef struct rocknpu_moe_experts_args {
    const int8_t * a8;          /* [tokens][hidden_pad], as rocknpu_hip_norm_a8 or rocknpu_hip_quantize_a8 give it; 16-byte aligned */
    const float * a_scales;     /* [tokens] */
    const int8_t * gate;        /* W8 [experts][ffn][hidden_pad]; 16-byte aligned, as up and down */
    const int8_t * up;          /* W8 [experts][ffn][hidden_pad] */
    const int8_t * down;        /* W8 [experts][hidden][ffn_pad] */
    const float * gate_scales;  /* [experts][ffn] */
    const float * up_scales;    /* [experts][ffn] */
    const float * down_scales;  /* [experts][hidden] */
    const int32_t * ids;        /* [tokens][top_k], as rocknpu_hip_moe_route gives them */
    const float * weights;      /* [tokens][top_k], its weights or others */
    const int32_t * plan;       /* the plan that came with the ids */
    void * out;                 /* [tokens][hidden] of out_type, rows out_row elements apart */
    int64_t tokens, out_row;    /* tokens * hidden_pad is below 2^32 */
    int32_t experts, top_k;
    int32_t hidden, hidden_pad; /* pads are multiples of 64, at most 133120, and what they add is zero in A8 or W8 */
    int32_t ffn, ffn_pad;
    uint32_t out_type;
} rocknpu_moe_experts_args;

/* The feed-forward of every token's chosen experts: for choice s of token t, on
 * expert e, g and u are the W8A8 products of the token's row with gate[e] and
 * up[e] (f32(f32(sum) * row's scale) * column's scale, as rocknpu_hip_gemm_w8a8),
 * v = f32(g * u / (1 + exp(-g))) with what is inside to 2^-50 of its value, v's row is
 * quantised as rocknpu_hip_quantize_a8 does, d is its product with down[e], and
 * out[t] = sum over s of weights[t][s] * d, in 64 bits in the order of s, rounded
 * to f32 and to out_type. Choices of id -1 are left out; a token without any gets zeros. A row of A8
 * whose scale is NaN gives NaN in its token's output and in no other.
 * out, the workspace and what the call reads overlap nowhere.
 * The workspace (rocknpu_hip_moe_experts_workspace bytes, 256-byte aligned, any
 * contents) is free again when the call's kernels are done. The same call gives
 * the same bits. */
int rocknpu_hip_moe_experts(const rocknpu_moe_experts_args * args, void * workspace, size_t workspace_bytes, void * stream);

/* Bytes of workspace for such a call (only its sizes are read). Host code only. */
int rocknpu_hip_moe_experts_workspace(const rocknpu_moe_experts_args * args, size_t * bytes);

/* How the gate and up product (gated = 1) or the down product of such a call (only its
 * sizes are read) is dealt out where the plan has `row_tiles` row tiles, on a GPU of
 * `cus` compute units (cus <= 0: the current device's). tile: its tiles' rows and output
 * columns, zeros where the call goes choice by choice. workgroups: those of the launch.
 * places, if not NULL, holds `capacity` entries of four words, one a workgroup: its row tile (-1: it
 * has none), its column tile, and which of how many parts of it: of one, of two (halves of the columns), of
 * four (0 and 1: those of the upper rows, 2 and 3: of the lower). A plan's first word is its row
 * tiles. Host code only. */
int rocknpu_hip_moe_product_places(const rocknpu_moe_experts_args * args, int gated, int32_t row_tiles, int cus,
                                   int32_t tile[2], int32_t * places, size_t capacity, size_t * workgroups);

#ifdef __cplusplus
}
#endif

#endif
