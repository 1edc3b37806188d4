// The experts' feed-forward of a few tokens (include/rocknpu_moe.h): two launches,
// each of which streams the chosen experts' weights once a choice.
//
// Bound by memory: a choice reads 3 * hidden * ffn bytes of weights for one row of
// products. v_mfma_i32_16x16x64_i8 takes 16 weight rows as its columns, lane l =
// 16 q + c supplying 16 bytes 64 i + 16 q of row c, so a wave's load is 16 runs of
// 64 bytes; the activation bytes are the same in all 16 rows of the other operand,
// of whose products row 0 is kept (lanes 0 - 15, first register). Sums over K are
// exact int32, so waves may share a row's K and add up in LDS.
//
// A token's output is worked out by one workgroup per 8 columns, which quantises
// the rows of all its choices itself: no launch for that, and none for the weighted
// sum. Its weights are asked for before. One token, top 8 of 64 experts of 2048 x 1024:
// 8.0 us gate and up (33.6 MB, 4.2 TB/s), 8.0 us down (16.8 MB; without the quantisation
// 1.5 us less, without the weights 5.7); by tiles, quantisation and sum 11 + 4 + 8 + 3.
// Top 2 of 8 of 4096 x 14336: 83 us in a graph, 4.2 TB/s.
#include "gemm_dma.h"
#include "moe_product.h"

namespace rk {
namespace {

constexpr int kGateWaves = 8;  // share a column tile's K
constexpr int kRing = 4;       // chunks of 64 bytes a wave asks for at once, of each matrix

__device__ __forceinline__ int row_of(const int32_t* ids, int at, int experts) {
    const int e = ids[at];
    return e < experts ? e : -1;
}

// SwiGLU's values of 16 columns of one choice, zeros behind ffn.
__global__ __launch_bounds__(kGateWaves * 64) void decode_gate_kernel(const MoeDecode p) {
    __shared__ int parts[2][kGateWaves][16];
    const int choice = blockIdx.x, c0 = blockIdx.y * 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, q = lane >> 4;
    const int e = row_of(p.ids, choice, p.experts);
    if (e < 0) return;
    const int token = choice / p.top_k, k = p.hidden_pad, chunks = k / 64;
    const int64_t row = static_cast<int64_t>(e) * p.ffn + min(c0 + col, p.ffn - 1);
    const int8_t* a = p.a + static_cast<int64_t>(token) * k + q * 16;
    const int8_t* w0 = p.gate + row * k + q * 16;
    const int8_t* w1 = p.up + row * k + q * 16;
    const float s0 = p.gate_scales[row], s1 = p.up_scales[row], as = p.a_scales[token];
    v4i g = {}, u = {};
    for (int i0 = wave; i0 < chunks; i0 += kGateWaves * kRing) {
        v4i av[kRing], gv[kRing], uv[kRing];
#pragma unroll
        for (int i = 0; i < kRing; ++i) {
            const int c = i0 + kGateWaves * i, at = min(c, chunks - 1) * 64;
            av[i] = *reinterpret_cast<const v4i*>(a + at);
            gv[i] = *reinterpret_cast<const v4i*>(w0 + at);
            uv[i] = *reinterpret_cast<const v4i*>(w1 + at);
        }
#pragma unroll
        for (int i = 0; i < kRing; ++i) {
            if (i0 + kGateWaves * i >= chunks) av[i] = v4i{};
            g = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[i], gv[i], g, 0, 0, 0);
            u = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[i], uv[i], u, 0, 0, 0);
        }
    }
    if (lane < 16) {
        parts[0][wave][lane] = g[0];
        parts[1][wave][lane] = u[0];
    }
    __syncthreads();
    if (threadIdx.x < 16) {
        int gs = 0, us = 0;
#pragma unroll
        for (int w = 0; w < kGateWaves; ++w) {
            gs += parts[0][w][col];
            us += parts[1][w][col];
        }
        const float v = swiglu((static_cast<float>(gs) * as) * s0, (static_cast<float>(us) * as) * s1);
        p.values[static_cast<int64_t>(choice) * p.ffn_pad + c0 + col] = c0 + col < p.ffn ? v : 0.0f;
    }
}

// A barrier for what is in LDS: a fenced one would wait for the weights' loads too.
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 8 columns of one token's output: the instruction's 16 columns are 8 weight rows
// twice, with one 64-byte chunk of K and with the next, and its rows 0 and 1 those
// chunks' codes, so loads are whole 128-byte lines and twice as many workgroups have
// work (16 columns: 11.7 us for 8 choices of 2048 x 1024). LDS: the codes of
// its choices' rows [top_k][ffn_pad] and 64 zeros, then the largest magnitudes' bits
// [top_k] and the sums [top_k][share][16]. `share` of the W waves take a choice's K together.
template <typename T, int W, int HOLD>
__global__ __launch_bounds__(W * 64) void decode_down_kernel(const MoeDecode p, int share, T* __restrict__ out, int64_t out_row) {
    extern __shared__ __align__(16) int8_t codes[];
    const int token = blockIdx.y, c0 = blockIdx.x * 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 7, second = lane >> 3 & 1, q = lane >> 4;
    const int k = p.ffn_pad, chunks = k / 64, pairs = (chunks + 1) / 2, n = p.top_k;
    uint32_t* peaks = reinterpret_cast<uint32_t*>(codes + static_cast<int64_t>(n) * k + 64);
    int* sums = reinterpret_cast<int*>(peaks + n);
    const int32_t* ids = p.ids + static_cast<int64_t>(token) * n;
    const int first = wave / share, part = wave % share, step = W / share;
    const int last_row = min(c0 + col, p.hidden - 1);
    constexpr int R = HOLD <= 2 ? kRing : 2 * kRing;  // pairs of chunks that a wave asks for at once
    v4i ring[R];
    const auto ask = [&](int s, int i0) {  // a wave's next chunks of choice s
        const int e = max(row_of(ids, min(s, n - 1), p.experts), 0);
        const int8_t* w = p.down + (static_cast<int64_t>(e) * p.hidden + last_row) * k + q * 16;
#pragma unroll
        for (int i = 0; i < R; ++i)
            ring[i] = *reinterpret_cast<const v4i*>(w + min(2 * (i0 + share * i) + second, chunks - 1) * 64);
    };
    const float* values = p.values + static_cast<int64_t>(token) * n * k;
    const int runs = (k + 255) / 256;
    const auto value = [&](int s, int run) {  // four values a lane
        return *reinterpret_cast<const float4*>(values + static_cast<int64_t>(s) * k + min(run * 256 + lane * 4, k - 4));
    };
    // The waves that share a choice's products share its row too, 256 values at a time,
    // and keep HOLD of their runs of the first choice in registers from the maximum to the
    // codes. Loads come back in the order in which they were asked for: these first, so
    // that they are quantised while the weights are on their way. Nothing here depends on
    // a condition that a wait would have to allow for: waves beyond the choices or the
    // runs do the last one's again. (A row that nothing was chosen for holds anything; its
    // codes and peak are not used.)
    const int mine = min(first, n - 1);
    const int own = min(static_cast<int>(threadIdx.x >> 3), n - 1);  // thread 8 s + c: choice s, column c
    const int own_e = row_of(ids, own, p.experts);
    float4 held[HOLD];
#pragma unroll
    for (int i = 0; i < HOLD; ++i) held[i] = value(mine, min(part + share * i, runs - 1));
    ask(first, part);
    const float own_weight = p.weights[static_cast<int64_t>(token) * n + own];
    const float own_scale = p.down_scales[static_cast<int64_t>(max(own_e, 0)) * p.hidden + last_row];
    if (threadIdx.x < n) peaks[threadIdx.x] = 0;
    int8_t* zeros = codes + static_cast<int64_t>(n) * k;
    if (threadIdx.x < 16) reinterpret_cast<int*>(zeros)[threadIdx.x] = 0;
    barrier();
    const auto peak_of = [&](int s, float4 v) {
        const uint32_t b = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                               max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
        const uint32_t peak = __float_as_uint(wave_max_nonneg(__uint_as_float(b)));
        if (lane == 0) atomicMax(&peaks[s], peak);
    };
    const auto quantise = [&](int s, int run, float4 v) {
        const uint32_t peak = peaks[s];
        const bool bad = peak > 0x7f7fffffu;
        const float scale = bad || peak == 0 ? 1.0f : __uint_as_float(peak) / 127.0f;
        const float x[4] = {v.x, v.y, v.z, v.w};
        uint32_t word[1];
        quant_sym_rcp_packed(x, scale, 1.0f / scale, scale >= 1.175494351e-38f, word);
        *reinterpret_cast<uint32_t*>(codes + static_cast<int64_t>(s) * k + min(run * 256 + lane * 4, k - 4)) = bad ? 0u : word[0];
    };
    const auto rest = [&](auto f) {  // the runs that are not held
        for (int s = first; s < n; s += step)
            for (int run = s == first ? part + share * HOLD : part; run < runs; run += share) f(s, run);
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i) peak_of(mine, held[i]);
    rest([&](int s, int run) { peak_of(s, value(s, run)); });
    barrier();
#pragma unroll
    for (int i = 0; i < HOLD; ++i) quantise(mine, min(part + share * i, runs - 1), held[i]);
    rest([&](int s, int run) { quantise(s, run, value(s, run)); });
    barrier();

    for (int s = first; s < n; s += step) {
        v4i acc = {};
        for (int i0 = part; i0 < pairs; i0 += share * R) {
            v4i w[R];
#pragma unroll
            for (int i = 0; i < R; ++i) w[i] = ring[i];
            const bool more = i0 + share * R < pairs;
            if (more || s + step < n) ask(more ? s : s + step, more ? i0 + share * R : part);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int c = 2 * (i0 + share * i) + (lane & 1);  // of the codes' row lane % 16: 0 or 1
                const v4i a = *reinterpret_cast<const v4i*>((c < chunks ? codes + static_cast<int64_t>(s) * k + c * 64 : zeros) + q * 16);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, w[i], acc, 0, 0, 0);
            }
        }
        if (lane < 16) sums[(s * share + part) * 16 + lane] = lane < 8 ? acc[0] : acc[1];
    }
    barrier();
    // the choices' values and weights side by side, in place of their sums (each thread
    // over what it alone has read); then they are added up one after the other, in 64
    // bits, where every product is exact
    float* terms = reinterpret_cast<float*>(sums);
    const auto term = [&](int s, float weight, float w_scale) {
        int total = 0;
        for (int j = 0; j < share; ++j) total += sums[(s * share + j) * 16 + col] + sums[(s * share + j) * 16 + 8 + col];
        const uint32_t peak = peaks[s];
        const float scale = peak > 0x7f7fffffu ? __builtin_nanf("") : peak == 0 ? 1.0f : __uint_as_float(peak) / 127.0f;
        terms[s * share * 16 + col] = (static_cast<float>(total) * scale) * w_scale;
        terms[s * share * 16 + 8 + col] = weight;
    };
    static_assert(8 * W >= ROCKNPU_MOE_MAX_TOP_K, "a thread for each choice's column");
    if (threadIdx.x < 8 * n) term(own, own_weight, own_scale);
    barrier();
    if (threadIdx.x < 8 && c0 + col < p.hidden) {
        double sum = 0.0;
        for (int s = 0; s < n; ++s)
            if (row_of(ids, s, p.experts) >= 0)
                sum += static_cast<double>(terms[s * share * 16 + 8 + col]) * static_cast<double>(terms[s * share * 16 + col]);
        out[token * out_row + c0 + col] = static_cast<T>(static_cast<float>(sum));
    }
}

constexpr int kDownWaves = 16;
int share_of(int top_k) { return top_k >= kDownWaves ? 1 : kDownWaves / top_k; }
size_t down_lds(int top_k, int ffn_pad) {
    return static_cast<size_t>(top_k) * ffn_pad + 64 + static_cast<size_t>(top_k) * 4 * (1 + 16 * share_of(top_k));
}

template <typename T>
int launch_down(const MoeDecode& p, void* out, int64_t out_row, hipStream_t stream) {
    const dim3 grid((p.hidden + 7) / 8, p.tokens), block(kDownWaves * 64);
    const int share = share_of(p.top_k), runs = (p.ffn_pad + 255) / 256;
    const size_t lds = down_lds(p.top_k, p.ffn_pad);
    if (runs <= 2 * share)
        decode_down_kernel<T, kDownWaves, 2><<<grid, block, lds, stream>>>(p, share, static_cast<T*>(out), out_row);
    else
        decode_down_kernel<T, kDownWaves, 8><<<grid, block, lds, stream>>>(p, share, static_cast<T*>(out), out_row);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

}  // namespace

// Whether a call goes choice by choice: one token's choices always, more tokens' while
// few of them fall on an expert that another has already called for (its weights are
// read again). By choices and by tiles, us in a graph: 64 experts of 2048 x 1024, top 8,
// of 1, 3, 4 and 8 tokens 16.4 and 23.2, 37.8 and 40.4, 48.6 and 45.8, 82 and 67; 8 of
// 4096 x 14336, top 2, of 1, 2 and 3: 83 and 117, 150 and 162, 215 and 194; 128 of 2048 x
// 768, top 8, of 3 and 4: 34.1 and 35.2, 42.0 and 40.6; 16 of 2048 x 5632, top 1, of 8
// and 12: 70 and 78, 97 and 84. The rows' codes have to fit LDS.
bool moe_decodes(int64_t tokens, int experts, int top_k, int ffn_pad) {
    const int64_t rows = tokens * top_k;
    return (tokens == 1 || (rows <= 28 && 2 * rows <= experts)) && down_lds(top_k, ffn_pad) <= 128 * 1024;
}

int launch_moe_decode(const MoeDecode& p, uint32_t out_type, void* out, int64_t out_row, hipStream_t stream) {
    const dim3 grid(p.tokens * p.top_k, p.ffn_pad / 16);
    decode_gate_kernel<<<grid, dim3(kGateWaves * 64), 0, stream>>>(p);
    if (hipGetLastError() != hipSuccess) return kStatusExec;
    return out_type == ROCKNPU_TYPE_F32   ? launch_down<float>(p, out, out_row, stream)
           : out_type == ROCKNPU_TYPE_F16 ? launch_down<_Float16>(p, out, out_row, stream)
                                          : launch_down<__bf16>(p, out, out_row, stream);
}

}  // namespace rk
