// The experts' products (include/rocknpu_moe.h): gate and up with SwiGLU, the
// rows' quantisation, down, and the weighted sum.
#include "moe.h"

#include <algorithm>
#include <climits>

namespace rk {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// One product over the plan's tiles: rows of `a` (of a token's choice: row / top_k,
// or of the choice's place itself) times the expert's matrices.
struct Product {
    const int8_t* a;
    const float* a_scales;
    const int8_t* w[2];
    const float* w_scales[2];
    float* out;
    int64_t ldo;
    int n, k, top_k;
};

__device__ __forceinline__ float swiglu(float g, float u) {
    const double x = static_cast<double>(g);
    return static_cast<float>(x * static_cast<double>(u) / (1.0 + exp(-x)));
}

// 64 x 64 tiles, a wave 32 x 32, operands straight from memory.
template <bool GATED>
__global__ __launch_bounds__(256) void product_kernel(const Product p, const MoePlan plan) {
    const int tiles = min(*plan.tile_count, plan.max_tiles);
    const int tile = blockIdx.x;
    if (tile >= tiles) return;
    const int e = min(max(plan.tiles[2 * tile], 0), plan.experts - 1);
    const int r0 = min(max(plan.tiles[2 * tile + 1], 0), plan.rows);
    const int end = min(min(plan.offsets[e + 1], plan.rows), r0 + plan.tile_rows);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int m0 = r0 + (wave & 1) * 32, n0 = blockIdx.y * 64 + (wave >> 1) * 32;
    if (m0 >= end || n0 >= p.n) return;
    const auto source = [&](int r) {
        r = min(r, end - 1);
        return GATED ? min(max(plan.order[r], 0), plan.rows - 1) / p.top_k : r;
    };
    const int8_t* a = p.a + static_cast<int64_t>(source(m0 + (lane & 31))) * p.k + half * 16;
    const int col = min(n0 + (lane & 31), p.n - 1);
    const int64_t wrow = static_cast<int64_t>(e) * p.n + col;
    const int8_t* w0 = p.w[0] + wrow * p.k + half * 16;
    const int8_t* w1 = GATED ? p.w[1] + wrow * p.k + half * 16 : nullptr;
    v16i acc[2] = {};
    for (int k = 0; k < p.k; k += 32) {
        const v4i av = *reinterpret_cast<const v4i*>(a + k);
        acc[0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, *reinterpret_cast<const v4i*>(w0 + k), acc[0], 0, 0, 0);
        if constexpr (GATED)
            acc[1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, *reinterpret_cast<const v4i*>(w1 + k), acc[1], 0, 0, 0);
    }
    const float s0 = p.w_scales[0][wrow], s1 = GATED ? p.w_scales[1][wrow] : 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = m0 + (i & 3) + 4 * half + 8 * (i >> 2);
        if (r >= end || n0 + (lane & 31) >= p.n) continue;
        const float as = p.a_scales[source(r)];
        float v = (static_cast<float>(acc[0][i]) * as) * s0;
        if constexpr (GATED) v = swiglu(v, (static_cast<float>(acc[1][i]) * as) * s1);
        p.out[static_cast<int64_t>(r) * p.ldo + n0 + (lane & 31)] = v;
    }
}

// out[t] = sum over the token's choices of weight * row.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ rows, const float* __restrict__ weights,
                                                      const MoePlan plan, int hidden, T* __restrict__ out, int64_t out_row) {
    const int t = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
    if (c >= hidden) return;
    float sum = 0.0f;
    for (int s = 0; s < plan.top_k; ++s) {
        const int i = t * plan.top_k + s, at = plan.place[i];
        if (at < 0 || at >= plan.rows) continue;
        sum += weights[i] * rows[static_cast<int64_t>(at) * hidden + c];
    }
    out[t * out_row + c] = static_cast<T>(sum);
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
size_t padded(size_t n) { return (n + 255) / 256 * 256; }

bool sizes_ok(const rocknpu_moe_experts_args* a) {
    return a && moe_size_ok(a->tokens, a->experts, a->top_k) && a->hidden >= 1 && a->hidden_pad >= a->hidden &&
           a->hidden_pad % 64 == 0 && a->hidden_pad <= kMaxExactK && a->ffn >= 1 && a->ffn_pad >= a->ffn &&
           a->ffn_pad % 64 == 0 && a->ffn_pad <= kMaxExactK;
}

// The workspace's parts: SwiGLU's rows, the down products in the same place; the
// quantised rows and their scales.
struct Space {
    size_t values, codes, scales;
    size_t bytes() const { return values + codes + scales; }
};
Space space(const rocknpu_moe_experts_args& a) {
    const size_t rows = static_cast<size_t>(a.tokens) * a.top_k;
    return {padded(rows * std::max(a.ffn, a.hidden) * 4), padded(rows * a.ffn_pad), padded(rows * 4)};
}

}  // namespace
}  // namespace rk

extern "C" int rocknpu_hip_moe_experts_workspace(const rocknpu_moe_experts_args* args, size_t* bytes) {
    using namespace rk;
    if (!bytes || !sizes_ok(args)) return kStatusInvalid;
    *bytes = space(*args).bytes();
    return kStatusOk;
}

extern "C" int rocknpu_hip_moe_experts(const rocknpu_moe_experts_args* args, void* workspace, size_t workspace_bytes,
                                       void* stream) {
    using namespace rk;
    if (!sizes_ok(args)) return kStatusInvalid;
    const rocknpu_moe_experts_args& a = *args;
    if (!a.gate || !a.up || !a.down || !a.gate_scales || !a.up_scales || !a.down_scales || !a.plan ||
        a.out_type > ROCKNPU_TYPE_BF16 || a.out_row < 0)
        return kStatusInvalid;
    if (!aligned(a.a8, 16) || !aligned(a.gate, 16) || !aligned(a.up, 16) || !aligned(a.down, 16) || !aligned(a.a_scales, 4) ||
        !aligned(a.gate_scales, 4) || !aligned(a.up_scales, 4) || !aligned(a.down_scales, 4) || !aligned(a.weights, 4) ||
        !aligned(a.plan, 4) || !aligned(a.out, a.out_type == ROCKNPU_TYPE_F32 ? 4 : 2))
        return kStatusInvalid;
    if (a.tokens > 1 && a.out_row < a.hidden) return kStatusInvalid;
    if (a.tokens == 0) return kStatusOk;
    const Space sp = space(a);
    if (!a.a8 || !a.a_scales || !a.weights || !a.out || !workspace || !aligned(workspace, 256) || workspace_bytes < sp.bytes())
        return kStatusInvalid;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const MoePlan plan = moe_plan(a.tokens, a.experts, a.top_k, const_cast<int32_t*>(a.plan), nullptr);
    uint8_t* at = static_cast<uint8_t*>(workspace);
    float* values = reinterpret_cast<float*>(at);
    int8_t* codes = reinterpret_cast<int8_t*>(at + sp.values);
    float* scales = reinterpret_cast<float*>(at + sp.values + sp.codes);
    const Product first{a.a8, a.a_scales, {a.gate, a.up}, {a.gate_scales, a.up_scales}, values, a.ffn, a.ffn, a.hidden_pad, a.top_k};
    product_kernel<true><<<dim3(plan.max_tiles, (a.ffn + 63) / 64), 256, 0, s>>>(first, plan);
    int st = launch_quantize_a8(values, plan.rows, a.ffn, a.ffn, a.ffn_pad, codes, scales, nullptr, 0, s);
    if (st != kStatusOk) return st;
    const Product second{codes, scales, {a.down, nullptr}, {a.down_scales, nullptr}, values, a.hidden, a.hidden, a.ffn_pad, a.top_k};
    product_kernel<false><<<dim3(plan.max_tiles, (a.hidden + 63) / 64), 256, 0, s>>>(second, plan);
    const dim3 grid(static_cast<unsigned>(a.tokens), (a.hidden + 255) / 256);
    if (a.out_type == ROCKNPU_TYPE_F32)
        combine_kernel<<<grid, 256, 0, s>>>(values, a.weights, plan, a.hidden, static_cast<float*>(a.out), a.out_row);
    else if (a.out_type == ROCKNPU_TYPE_F16)
        combine_kernel<<<grid, 256, 0, s>>>(values, a.weights, plan, a.hidden, static_cast<_Float16*>(a.out), a.out_row);
    else
        combine_kernel<<<grid, 256, 0, s>>>(values, a.weights, plan, a.hidden, static_cast<__bf16*>(a.out), a.out_row);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}
