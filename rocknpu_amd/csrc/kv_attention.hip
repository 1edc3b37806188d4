// Attention over the 8-bit key/value cache (include/rocknpu_kv.h).
#include <algorithm>
#include <climits>

#include "kv.h"

namespace rk {
namespace {

struct AttentionParams {
    rocknpu_kv_cache c;
    rocknpu_kv_attention_args a;
    float* state;  // [rows][heads][2]: running maximum and sum, for the block weights
};

// A page's scale, NaN where there is none or it is not finite.
__device__ __forceinline__ float kv_scale(const rocknpu_kv_cache& c, int64_t page, int which, bool ok) {
    const float s = ok ? c.scales[2 * page + which] : 0.0f;
    return ok && fabsf(s) <= 3.402823466e38f ? s : __builtin_nanf("");
}

// The score of one key after scale, cap, bias and mask.
__device__ __forceinline__ float masked_score(const rocknpu_kv_attention_args& a, float dot, int head, int kpos, int qpos,
                                              int total, int prefix) {
    float x = a.scale * dot;
    if (a.softcap != 0.0f) x = a.softcap * tanhf(x / a.softcap);
    if (a.slopes) x += a.slopes[head] * static_cast<float>(kpos - qpos);
    bool seen = !a.causal || (kpos <= qpos && (a.window == 0 || kpos > qpos - a.window));
    seen |= kpos < prefix;
    return seen && kpos < total ? x : -__builtin_inff();
}

// One wave per query row and head; lane l holds token l % 32 of a block for the
// scores (its half of the dims), and dims l, l + 64, .. for the output.
template <int TYPE, int D>
__global__ __launch_bounds__(64) void kv_attention_kernel(AttentionParams p) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    __shared__ float q[D];
    const rocknpu_kv_cache& c = p.c;
    const rocknpu_kv_attention_args& a = p.a;
    const int lane = threadIdx.x, b = blockIdx.z, head = blockIdx.y, i = blockIdx.x;
    const KvSpan s = kv_span(a.past, a.cu, b, static_cast<int>(a.rows), static_cast<int>(a.max_new));
    if (i >= s.n) return;
    const int total = s.past + s.n, qpos = s.past + i, h = head / (a.heads / c.kv_heads);
    const int held = min((total + kKvBlock - 1) / kKvBlock - max(c.dropped[b], 0), c.max_blocks);
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const int64_t entry_row = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks;
    const T* qr = static_cast<const T*>(a.q) + (s.row0 + i) * a.q_row + head * a.q_head;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) q[lane + 64 * e] = K::to_f32(qr[lane + 64 * e]);
    __syncthreads();
    float top = -__builtin_inff(), sum = 0.0f, o[D / 64] = {};
    const int t = lane & 31, half = lane >> 5;
    for (int at = 0; at < held; ++at) {
        const int page = c.table[entry_row + at];
        const bool ok = page >= 0 && page < c.n_pages;
        const int64_t pg = ok ? page : 0;
        const int8_t* keys = reinterpret_cast<const int8_t*>(c.pages) + pg * (2 * kKvBlock * D);
        const int8_t* values = keys + kKvBlock * D;
        const float sk = kv_scale(c, pg, 0, ok), sv = kv_scale(c, pg, 1, ok);
        float dot = 0.0f;
        for (int e = 0; e < D / 2; ++e) {
            const int d = half * (D / 2) + e;
            dot += q[d] * static_cast<float>(keys[kv_key_at(t, d)]);
        }
        dot += __shfl_xor(dot, 32, 64);
        const float x = masked_score(a, dot * sk, head, c.starts[entry_row + at] + t, qpos, total, prefix);
        const float m = fmaxf(top, wave_max(x));
        const bool any = __any(x != -__builtin_inff());  // a NaN counts
        if (!any) continue;
        const float w = x == -__builtin_inff() ? 0.0f : expf(x - m);
        const float keep = top == -__builtin_inff() ? 0.0f : expf(top - m);
        float l = half ? 0.0f : w;
#pragma unroll
        for (int g = 32; g >= 1; g >>= 1) l += __shfl_xor(l, g, 64);
        sum = sum * keep + l;
        top = m;
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[e] *= keep;
        for (int k = 0; k < kKvBlock; ++k) {
            const float wk = __shfl(w, k, 64);
            if (wk == 0.0f) continue;
#pragma unroll
            for (int e = 0; e < D / 64; ++e)
                o[e] += wk * (static_cast<float>(values[kv_value_at(k, lane + 64 * e)]) * sv);
        }
    }
    T* out = static_cast<T*>(a.out) + (s.row0 + i) * a.out_row + head * a.out_head;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) out[lane + 64 * e] = K::from_f32(sum == 0.0f ? 0.0f : o[e] / sum);
    if (p.state && lane == 0) {
        float* st = p.state + 2 * (static_cast<int64_t>(s.row0 + i) * a.heads + head);
        st[0] = top;
        st[1] = sum;
    }
}

// One wave per block of a sequence and kv head: the scores of its rows again,
// with their final maximum and sum.
template <int TYPE, int D>
__global__ __launch_bounds__(64) void kv_weights_kernel(AttentionParams p) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    __shared__ float q[D];
    const rocknpu_kv_cache& c = p.c;
    const rocknpu_kv_attention_args& a = p.a;
    const int lane = threadIdx.x, b = blockIdx.z, h = blockIdx.y, at = blockIdx.x;
    const KvSpan s = kv_span(a.past, a.cu, b, static_cast<int>(a.rows), static_cast<int>(a.max_new));
    const int total = s.past + s.n, group = a.heads / c.kv_heads;
    const int held = min((total + kKvBlock - 1) / kKvBlock - max(c.dropped[b], 0), c.max_blocks);
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const int64_t entry = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks + at;
    float got = 0.0f;
    if (at < held) {
        const int page = c.table[entry];
        const bool ok = page >= 0 && page < c.n_pages;
        const int64_t pg = ok ? page : 0;
        const int8_t* keys = reinterpret_cast<const int8_t*>(c.pages) + pg * (2 * kKvBlock * D);
        const float sk = kv_scale(c, pg, 0, ok);
        const int t = lane & 31, half = lane >> 5;
        for (int r = 0; r < s.n * group; ++r) {
            const int i = r / group, head = h * group + r % group;
            const T* qr = static_cast<const T*>(a.q) + (s.row0 + i) * a.q_row + head * a.q_head;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < D / 64; ++e) q[lane + 64 * e] = K::to_f32(qr[lane + 64 * e]);
            __syncthreads();
            float dot = 0.0f;
            for (int e = 0; e < D / 2; ++e) {
                const int d = half * (D / 2) + e;
                dot += q[d] * static_cast<float>(keys[kv_key_at(t, d)]);
            }
            dot += __shfl_xor(dot, 32, 64);
            const float x = masked_score(a, dot * sk, head, c.starts[entry] + t, s.past + i, total, prefix);
            const float* st = p.state + 2 * (static_cast<int64_t>(s.row0 + i) * a.heads + head);
            float l = half || x == -__builtin_inff() ? 0.0f : expf(x - st[0]) / st[1];
#pragma unroll
            for (int g = 32; g >= 1; g >>= 1) l += __shfl_xor(l, g, 64);
            got += l;
        }
    }
    if (lane == 0) a.weights_out[entry] = c.weights[entry] + got;
}

template <int TYPE, int D>
int launch(const AttentionParams& p, hipStream_t stream) {
    const rocknpu_kv_attention_args& a = p.a;
    if (a.rows > 0 && a.max_new > 0)
        kv_attention_kernel<TYPE, D><<<dim3(static_cast<unsigned>(a.max_new), a.heads, p.c.batch), 64, 0, stream>>>(p);
    if (a.weights_out)
        kv_weights_kernel<TYPE, D><<<dim3(p.c.max_blocks, p.c.kv_heads, p.c.batch), 64, 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <int TYPE>
int launch_dim(const AttentionParams& p, hipStream_t stream) {
    switch (p.c.head_dim) {
        case 64: return launch<TYPE, 64>(p, stream);
        case 128: return launch<TYPE, 128>(p, stream);
        case 192: return launch<TYPE, 192>(p, stream);
        default: return launch<TYPE, 256>(p, stream);
    }
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// What the host can see of a call.
bool attention_ok(const rocknpu_kv_cache* c, const rocknpu_kv_attention_args* a) {
    if (!kv_cache_ok(c) || !a || a->type > ROCKNPU_KV_BF16) return false;
    if (a->rows < 0 || a->rows > INT_MAX || a->max_new < 0 || a->max_new > INT_MAX || a->max_tokens < 0) return false;
    if (a->heads < 1 || a->heads > 65535 || a->heads % c->kv_heads != 0 || a->window < 0) return false;
    if (!a->causal && (a->window != 0 || a->prefix)) return false;
    if (!(a->scale - a->scale == 0.0f) || !(a->softcap >= 0.0f) || !(a->softcap - a->softcap == 0.0f)) return false;
    if (!a->past || !a->cu) return false;
    const int size = a->type == ROCKNPU_KV_F32 ? 4 : 2;
    if (a->rows > 0 && (!a->q || !a->out)) return false;
    if (!aligned(a->q, size) || !aligned(a->out, size) || a->q_row < 0 || a->q_head < 0 || a->out_row < 0 || a->out_head < 0)
        return false;
    if (a->weights_out && (!c->weights || a->max_new * (a->heads / c->kv_heads) > kKvMaxWeightRows)) return false;
    return true;
}

size_t attention_bytes(const rocknpu_kv_attention_args& a) {
    return a.weights_out ? (static_cast<size_t>(a.rows) * a.heads * 8 + 255) / 256 * 256 : 0;
}

}  // namespace
}  // namespace rk

extern "C" int rocknpu_hip_kv_attention_workspace(const rocknpu_kv_cache* cache, const rocknpu_kv_attention_args* args,
                                                  int cus, size_t* bytes) {
    using namespace rk;
    if (!bytes || !attention_ok(cache, args)) return kStatusInvalid;
    (void)cus;
    *bytes = attention_bytes(*args);
    return kStatusOk;
}

extern "C" int rocknpu_hip_kv_attention(const rocknpu_kv_cache* cache, const rocknpu_kv_attention_args* args,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    using namespace rk;
    if (!attention_ok(cache, args)) return kStatusInvalid;
    const size_t need = attention_bytes(*args);
    if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) return kStatusInvalid;
    if ((args->rows == 0 || args->max_new == 0) && !args->weights_out) return kStatusOk;
    AttentionParams p{*cache, *args, need ? static_cast<float*>(workspace) : nullptr};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (args->type) {
        case ROCKNPU_KV_F32: return launch_dim<ROCKNPU_KV_F32>(p, s);
        case ROCKNPU_KV_F16: return launch_dim<ROCKNPU_KV_F16>(p, s);
        default: return launch_dim<ROCKNPU_KV_BF16>(p, s);
    }
}
