// The experts' products (include/rocknpu_moe.h): gate and up with SwiGLU, the
// rows' quantisation, down, and the weighted sum.
#include "moe_product.h"

#include <algorithm>
#include <climits>

namespace rk {
namespace {

// out[t] = sum over the token's choices, in their order, of weight * row, in 64 bits
// (where every product is exact), rounded to f32 and to out's type. Bound by
// memory: top_k rows are read for each that is written (32768 rows of 2048 in 51 us,
// 5.9 TB/s). A thread takes 4 columns of a token and asks for four choices' rows
// before it adds them up. Rows are ld floats apart, a multiple of 4; VEC: out's
// columns can be stored four at a time.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ rows, int ld, const float* __restrict__ weights,
                                                      const int32_t* __restrict__ place, int top_k, int hidden, int n_rows,
                                                      T* __restrict__ out, int64_t out_row) {
    typedef float vec __attribute__((ext_vector_type(4)));
    const int64_t t = blockIdx.x;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 4;
    if (c >= hidden) return;
    place += t * top_k;
    weights += t * top_k;
    double sum[4] = {};
    for (int s0 = 0; s0 < top_k; s0 += 4) {
        vec v[4];
        float w[4];
        bool used[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = min(s0 + i, top_k - 1), at = place[s];
            used[i] = s0 + i < top_k && at >= 0 && at < n_rows;
            w[i] = weights[s];
            v[i] = *reinterpret_cast<const vec*>(rows + static_cast<int64_t>(used[i] ? at : 0) * ld + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (used[i])
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += static_cast<double>(w[i]) * static_cast<double>(v[i][e]);
    }
    struct alignas(sizeof(T) * 4) Out {
        T e[4];
    } o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.e[e] = static_cast<T>(static_cast<float>(sum[e]));
    T* y = out + t * out_row + c;
    if constexpr (VEC) {
        *reinterpret_cast<Out*>(y) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < hidden) y[e] = o.e[e];
    }
}

template <typename T>
int launch_combine(const float* rows, int ld, const float* weights, const MoePlan& plan, int64_t tokens, int hidden, void* out,
                   int64_t out_row, hipStream_t stream) {
    T* o = static_cast<T*>(out);
    const int cols = ld / 4, nt = std::min(256, (cols + 63) / 64 * 64);
    const dim3 grid(static_cast<unsigned>(tokens), (cols + nt - 1) / nt);
    if (hidden % 4 == 0 && out_row % 4 == 0 && reinterpret_cast<uintptr_t>(o) % (4 * sizeof(T)) == 0)
        combine_kernel<T, true><<<grid, nt, 0, stream>>>(rows, ld, weights, plan.place, plan.top_k, hidden, plan.rows, o, out_row);
    else
        combine_kernel<T, false><<<grid, nt, 0, stream>>>(rows, ld, weights, plan.place, plan.top_k, hidden, plan.rows, o, out_row);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
size_t padded(size_t n) { return (n + 255) / 256 * 256; }

bool sizes_ok(const rocknpu_moe_experts_args* a) {
    return a && moe_size_ok(a->tokens, a->experts, a->top_k) && a->hidden >= 1 && a->hidden_pad >= a->hidden &&
           a->hidden_pad % 64 == 0 && a->hidden_pad <= kMaxExactK && a->ffn >= 1 && a->ffn_pad >= a->ffn &&
           a->ffn_pad % 64 == 0 && a->ffn_pad <= kMaxExactK &&
           a->tokens <= INT64_C(0xffffffff) / a->hidden_pad;  // offsets into A8 are 32 bits
}

// The workspace's parts: SwiGLU's rows, the down products in the same place; the
// quantised rows and their scales.
struct Space {
    size_t values, codes, scales;
    size_t bytes() const { return values + codes + scales; }
};
Space space(const rocknpu_moe_experts_args& a) {
    const size_t rows = static_cast<size_t>(a.tokens) * a.top_k;
    return {padded(rows * std::max(a.ffn_pad, (a.hidden + 3) / 4 * 4) * 4), padded(rows * a.ffn_pad), padded(rows * 4)};
}

}  // namespace
}  // namespace rk

extern "C" int rocknpu_hip_moe_experts_workspace(const rocknpu_moe_experts_args* args, size_t* bytes) {
    using namespace rk;
    if (!bytes || !sizes_ok(args)) return kStatusInvalid;
    *bytes = space(*args).bytes();
    return kStatusOk;
}

extern "C" int rocknpu_hip_moe_product_places(const rocknpu_moe_experts_args* args, int gated, int32_t row_tiles, int cus,
                                              int32_t tile[2], int32_t* places, size_t capacity, size_t* workgroups) {
    using namespace rk;
    if (!tile || !workgroups || !sizes_ok(args)) return kStatusInvalid;
    const MoePlan plan = moe_plan(args->tokens, args->experts, args->top_k, nullptr, nullptr);
    if (row_tiles < 0 || row_tiles > plan.max_tiles) return kStatusInvalid;
    tile[0] = tile[1] = 0;
    *workgroups = 0;
    if (args->tokens == 0 || moe_decodes(args->tokens, args->experts, args->top_k, args->ffn_pad)) return kStatusOk;
    const int n = gated ? args->ffn : args->hidden, xcd_cus = moe_xcd_cus(cus > 0 ? cus : device_cu_count());
    tile[0] = plan.tile_rows;
    tile[1] = moe_tile_columns(plan.tile_rows, gated != 0);
    *workgroups = static_cast<size_t>(moe_product_grid(plan, n, gated != 0, xcd_cus));
    if (!places) return kStatusOk;
    if (*workgroups > 0x7fffffff || capacity < *workgroups) return kStatusInvalid;
    for (size_t b = 0; b < *workgroups; ++b) {
        const MoeShare share = moe_share(b & 7, row_tiles, (n + tile[1] - 1) / tile[1], xcd_cus, plan.tile_rows == 256);
        int32_t* p = places + 4 * b;
        int i = static_cast<int>(b >> 3);
        moe_part(share, i, p[2]);
        p[0] = -1;
        p[1] = 0;
        if (i < share.mine) moe_pair(share, i, p[0], p[1]);
        p[3] = moe_splits(share, i) ? share.parts : 1;
    }
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
        !aligned(a.gate_scales, 4) || !aligned(a.up_scales, 4) || !aligned(a.down_scales, 4) || !aligned(a.ids, 4) || !aligned(a.weights, 4) ||
        !aligned(a.plan, 4) || !aligned(a.out, a.out_type == ROCKNPU_TYPE_F32 ? 4 : 2))
        return kStatusInvalid;
    if (a.tokens > 1 && a.out_row < a.hidden) return kStatusInvalid;
    if (a.tokens == 0) return kStatusOk;
    const Space sp = space(a);
    if (!a.a8 || !a.a_scales || !a.ids || !a.weights || !a.out || !workspace || !aligned(workspace, 256) || workspace_bytes < sp.bytes())
        return kStatusInvalid;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const MoePlan plan = moe_plan(a.tokens, a.experts, a.top_k, const_cast<int32_t*>(a.plan), nullptr);
    uint8_t* at = static_cast<uint8_t*>(workspace);
    float* values = reinterpret_cast<float*>(at);
    int8_t* codes = reinterpret_cast<int8_t*>(at + sp.values);
    float* scales = reinterpret_cast<float*>(at + sp.values + sp.codes);
    if (moe_decodes(a.tokens, a.experts, a.top_k, a.ffn_pad)) {
        const MoeDecode d{a.a8, a.a_scales, a.gate, a.up, a.down, a.gate_scales, a.up_scales, a.down_scales, a.ids, a.weights,
                          values, static_cast<int>(a.tokens), a.experts, a.top_k, a.hidden, a.hidden_pad, a.ffn, a.ffn_pad};
        return launch_moe_decode(d, a.out_type, a.out, a.out_row, s);
    }
    // rows of whole 16 bytes, so that what reads them can
    const int values_row = (a.ffn + 63) / 64 * 64, out_row = (a.hidden + 3) / 4 * 4;
    const MoeProduct first{a.a8, a.a_scales, {a.gate, a.up}, {a.gate_scales, a.up_scales}, values, a.ffn, a.hidden_pad, values_row, a.top_k};
    int st = launch_moe_product(first, true, plan, s);
    if (st != kStatusOk) return st;
    constexpr int kRowsOnce = 1 << 21;  // a launch holds less than 2^32 threads, a row up to 1024
    for (int r = 0; r < plan.rows; r += kRowsOnce) {
        st = launch_quantize_a8(values + static_cast<size_t>(r) * values_row, std::min(plan.rows - r, kRowsOnce), values_row, values_row,
                                a.ffn_pad, codes + static_cast<size_t>(r) * a.ffn_pad, scales + r, nullptr, 0, s);
        if (st != kStatusOk) return st;
    }
    const MoeProduct second{codes, scales, {a.down, nullptr}, {a.down_scales, nullptr}, values, a.hidden, a.ffn_pad, out_row, a.top_k};
    st = launch_moe_product(second, false, plan, s);
    if (st != kStatusOk) return st;
    if (a.out_type == ROCKNPU_TYPE_F32) return launch_combine<float>(values, out_row, a.weights, plan, a.tokens, a.hidden, a.out, a.out_row, s);
    if (a.out_type == ROCKNPU_TYPE_F16) return launch_combine<_Float16>(values, out_row, a.weights, plan, a.tokens, a.hidden, a.out, a.out_row, s);
    return launch_combine<__bf16>(values, out_row, a.weights, plan, a.tokens, a.hidden, a.out, a.out_row, s);
}
