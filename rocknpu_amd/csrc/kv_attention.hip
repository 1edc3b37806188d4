// Attention over the 8-bit key/value cache (include/rocknpu_kv.h).
#include <algorithm>
#include <climits>

#include "kv_attend.h"

namespace rk {
namespace {

struct AttentionParams {
    rocknpu_kv_cache c;
    rocknpu_kv_attention_args a;
};

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
        const float sk = kv_scale(c.scales[2 * pg], ok), sv = kv_scale(c.scales[2 * pg + 1], ok);
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
}

template <int TYPE, int D>
int launch(const AttentionParams& p, hipStream_t stream) {
    const rocknpu_kv_attention_args& a = p.a;
    kv_attention_kernel<TYPE, D><<<dim3(static_cast<unsigned>(a.max_new), a.heads, p.c.batch), 64, 0, stream>>>(p);
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

size_t padded(size_t n) { return (n + 255) / 256 * 256; }

// Rows of a kv head up to which the cache is streamed through 16-row tiles.
constexpr int64_t kStreamRows = 32;
// Blocks of a split, at least: two for each of a workgroup's waves.
constexpr int kMinChunk = 8;
// Sequences up to which their blocks are shared out over the workgroups.
constexpr int kMaxShared = 1024;

struct Plan {
    KvAttend p;
    bool stream;
    size_t out_bytes, state_bytes, sums_bytes;
    size_t bytes() const { return out_bytes + state_bytes + sums_bytes; }
};

Plan plan(const rocknpu_kv_cache& c, const rocknpu_kv_attention_args& a, int cus) {
    Plan r{};
    KvAttend& p = r.p;
    p.c = c;
    p.a = a;
    p.group = a.heads / c.kv_heads;
    const int64_t per = a.type == ROCKNPU_KV_F32 ? 4 : 8;
    p.vec_q = aligned(a.q, 16) && a.q_row % per == 0 && a.q_head % per == 0;
    p.vec_out = aligned(a.out, 16) && a.out_row % per == 0 && a.out_head % per == 0;
    const int64_t rows = std::max<int64_t>(a.max_new, 1) * p.group;
    r.stream = rows <= kStreamRows || a.weights_out;
    if (!r.stream) return r;
    p.row_tiles = static_cast<int>((rows + kKvTileRows - 1) / kKvTileRows);
    int64_t blocks = a.max_tokens > 0 ? (a.max_tokens + kKvBlock - 1) / kKvBlock : c.max_blocks;
    if (a.window > 0) blocks = std::min<int64_t>(blocks, (static_cast<int64_t>(a.window) + a.max_new) / kKvBlock + 2);
    blocks = std::max<int64_t>(1, std::min<int64_t>(blocks, c.max_blocks));
    p.min_chunk = kMinChunk;
    // One round of the workgroups that the GPU holds at once: a second round pays every workgroup's start (lookups, the
    // queries, the first blocks' latency) again. Sharing rounds each sequence up, by half a workgroup on average. 32
    // ragged sequences of 500-4100 tokens, 8 kv heads of 128: 40.4 us; three quarters and one and a half rounds 48.7
    // and 47.3; a fixed four parts a sequence 51.4.
    const int64_t resident = (c.head_dim <= 64 ? 3 : c.head_dim <= 128 ? 2 : 1) * cus;
    const int64_t share = std::max<int64_t>(resident / (c.kv_heads * p.row_tiles) - c.batch / 2, 1);
    const bool shared = blocks > p.min_chunk && c.batch <= kMaxShared && rows > 0;
    p.share = shared ? static_cast<int>(std::min<int64_t>(share, c.batch * ((blocks + p.min_chunk - 1) / p.min_chunk))) : 0;
    p.slots = p.share + c.batch;
    const size_t slots = static_cast<size_t>(p.slots) * c.kv_heads * p.row_tiles * kKvTileRows;
    if (p.share) r.out_bytes = padded(slots * c.head_dim * 4);
    if (p.share || a.weights_out) r.state_bytes = padded(slots * 8);
    if (a.weights_out)
        r.sums_bytes = padded(static_cast<size_t>(c.batch) * c.kv_heads * c.max_blocks * p.row_tiles * kKvTileRows * 8);
    return r;
}

}  // namespace
}  // namespace rk

extern "C" int rocknpu_hip_kv_attention_workspace(const rocknpu_kv_cache* cache, const rocknpu_kv_attention_args* args,
                                                  int cus, size_t* bytes) {
    using namespace rk;
    if (!bytes || !attention_ok(cache, args)) return kStatusInvalid;
    *bytes = plan(*cache, *args, cus > 0 ? cus : device_cu_count()).bytes();
    return kStatusOk;
}

extern "C" int rocknpu_hip_kv_attention(const rocknpu_kv_cache* cache, const rocknpu_kv_attention_args* args,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    using namespace rk;
    if (!attention_ok(cache, args)) return kStatusInvalid;
    Plan r = plan(*cache, *args, device_cu_count());
    const size_t need = r.bytes();
    if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) return kStatusInvalid;
    if ((args->rows == 0 || args->max_new == 0) && !args->weights_out) return kStatusOk;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (r.stream) {
        uint8_t* at = static_cast<uint8_t*>(workspace);
        if (r.out_bytes) r.p.part_out = reinterpret_cast<float*>(at);
        if (r.state_bytes) r.p.part_state = reinterpret_cast<float*>(at + r.out_bytes);
        if (r.sums_bytes) r.p.block_sums = reinterpret_cast<float*>(at + r.out_bytes + r.state_bytes);
        return launch_kv_stream(r.p, s);
    }
    AttentionParams p{*cache, *args};
    switch (args->type) {
        case ROCKNPU_KV_F32: return launch_dim<ROCKNPU_KV_F32>(p, s);
        case ROCKNPU_KV_F16: return launch_dim<ROCKNPU_KV_F16>(p, s);
        default: return launch_dim<ROCKNPU_KV_BF16>(p, s);
    }
}
