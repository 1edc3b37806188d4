// Root-mean-square norm with the residual's addition in front of it and the
// symmetric int8 quantisation of its rows behind it: what stands between the
// output of one projection and the A8 rows of the next. No counterpart in the
// reference's accelerated path (its LLM glue norms on the host,
// crates/rocknpu-llm/src/lib.rs; the quantisation is quant.hip's,
// crates/rocknpu-capi/src/lib.rs:614-654).
//
// h = f32(x) + f32(r), hidden = round(h), u = h * w in f32,
// s0 = max|u| / 127 (1 for a zero row), codes = round_half_away(u / s0),
// f = 1 / sqrt(mean(h^2) + eps), scale = s0 * f, out = round(u * f).
// f multiplies the whole row, so the codes need no f: they are u's, exact to
// the bit whatever order the sum of squares has, and quantising needs the row's
// largest |u| alone. f itself is worked out in 64 bits, the squares' sum included
// (f32 partial sums of up to 64 squares a thread lose bits where one channel is far above
// the others, as in residual streams: rms error of the scale 5.9e-8 at 16384 columns
// where its rounding alone is 2.0e-8), so the scale has one rounding.
//
// Bound by memory: a row is read once, into registers, and everything is written
// from them, up to 32768 columns, 16384 where no wide loads fit. The compiler keeps a part
// of longer rows in memory (336 to 432 bytes a lane, and 760 to 772), and they run
// at a fraction of the rate: 1024 rows of 32768 f32 94 us, 4.7 TB/s, of 65536 400 us, 2.2;
// bf16 46 us, 5.2, and 289, 1.6; 65535 f16 1145 us, 0.4. One workgroup a row. With a residual (x and r read, hidden and codes
// written), in a graph: 16384 rows of 4096 f32 152 us, 5.7 TB/s, bf16 88 us, 5.4; of
// 1024 f32 35 us, 6.3; 16384 rows of 64 f32 8 us; one row of 2048 3.3 us.
#include "common.h"
#include "rocknpu_hip.h"

#include <algorithm>
#include <climits>

namespace rk {
namespace {

template <typename T, int V>
struct alignas(sizeof(T) * V) Run {
    T e[V];
};

// Sum over the wave in 64 bits: DPP steps within rows of 16 lanes, then the four
// rows by lane reads. Every lane gets the result.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xF, 0xF, true);
    return v + __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}
__device__ __forceinline__ double read_lane(double v, int lane) {
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
    return __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}
__device__ __forceinline__ double wave_sum(double v) {
    v = dpp_add<0xB1>(v);   // lanes 1 0 3 2
    v = dpp_add<0x4E>(v);   // lanes 2 3 0 1
    v = dpp_add<0x141>(v);  // mirrored within 8
    v = dpp_add<0x140>(v);  // mirrored within 16
    return (read_lane(v, 0) + read_lane(v, 16)) + (read_lane(v, 32) + read_lane(v, 48));
}

// Thread t of nt holds R runs of V values, run t + nt j of its row. V > 1: k, the
// strides and the bases allow whole runs as one load; V = 1: any (16384 rows of
// 2047 f32 90 us, 4.9 TB/s, f16 85, 2.8; runs of 16 bytes with 4- or 2-byte alignment
// and the last one in parts took 106 and 71, and 1000 rows of f16 8.5 against 6.9).
template <typename T, typename W, int V, int R>
__global__ __launch_bounds__(1024) void norm_a8_kernel(const T* x, const T* r, const W* __restrict__ weight,
                                                       int64_t x_row, int64_t r_row, int k, int nt, T* hidden,
                                                       int64_t hidden_row, T* out, int64_t out_row,
                                                       int8_t* __restrict__ a8, int64_t k_pad,
                                                       float* __restrict__ scales, float eps) {
    constexpr int N = V * R;
    __shared__ uint32_t red_max[16];
    __shared__ double red_sum[16];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, runs = k / V;
    Run<T, V> xv[R], rv[R];
    Run<W, V> wv[R];
    const Run<T, V>* xr = reinterpret_cast<const Run<T, V>*>(x + row * x_row);
    const Run<T, V>* rr = reinterpret_cast<const Run<T, V>*>(r + row * r_row);
    const Run<W, V>* wr = reinterpret_cast<const Run<W, V>*>(weight);
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = t + nt * j;
        xv[j] = Run<T, V>{};
        rv[j] = Run<T, V>{};
        wv[j] = Run<W, V>{};
        if (i < runs) {
            xv[j] = xr[i];
            if (r) rv[j] = rr[i];
            wv[j] = wr[i];
        }
    }
    float u[N];
    double sum = 0.0;
    uint32_t um = 0;
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float a = static_cast<float>(xv[j].e[e]);
            const float h = r ? a + static_cast<float>(rv[j].e[e]) : a;
            u[V * j + e] = h;
            sum = fma(static_cast<double>(h), static_cast<double>(h), sum);
        }
    if (hidden) {
        Run<T, V>* hr = reinterpret_cast<Run<T, V>*>(hidden + row * hidden_row);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int i = t + nt * j;
            Run<T, V> v;
#pragma unroll
            for (int e = 0; e < V; ++e) v.e[e] = static_cast<T>(u[V * j + e]);
            if (i < runs) hr[i] = v;
        }
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int i = V * j + e;
            u[i] = u[i] * static_cast<float>(wv[j].e[e]);
            um = max(um, __float_as_uint(u[i]) & 0x7fffffffu);
        }
    um = __float_as_uint(wave_max_nonneg(__uint_as_float(um)));
    sum = wave_sum(sum);
    if (nt > 64) {
        if ((t & 63) == 0) {
            red_max[t >> 6] = um;
            red_sum[t >> 6] = sum;
        }
        __syncthreads();
        um = red_max[0];
        sum = red_sum[0];
        for (int w = 1; w < nt / 64; ++w) {
            um = max(um, red_max[w]);
            sum += red_sum[w];
        }
    }
    const bool bad = um > 0x7f7fffffu;  // a value that is not finite
    const float peak = __uint_as_float(um);
    const float step = bad || peak == 0.0f ? 1.0f : peak / 127.0f;
    const float inv = 1.0f / step;
    int8_t* q = a8 + row * k_pad;
    if constexpr (N % 4 == 0 && V > 1) {
        uint32_t w[N / 4];
        quant_sym_rcp_packed(u, step, inv, step >= 1.175494351e-38f, w);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int i = t + nt * j;
            if (i < runs) {
                if constexpr (V == 8)
                    reinterpret_cast<uint2*>(q)[i] = bad ? uint2{0, 0} : uint2{w[2 * j], w[2 * j + 1]};
                else
                    reinterpret_cast<uint32_t*>(q)[i] = bad ? 0u : w[j];
            }
        }
    } else {
        int c[N];
        quant_sym_rcp(u, step, inv, c);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int i = t + nt * j;
            if (i < runs) q[i] = bad ? 0 : static_cast<int8_t>(c[j]);
        }
    }
    for (int64_t i = k + t; i < k_pad; i += nt) q[i] = 0;
    if (out || t == 0) {
        const double f = bad ? __builtin_nan("") : 1.0 / sqrt(sum / static_cast<double>(k) + static_cast<double>(eps));
        if (t == 0) scales[row] = static_cast<float>(static_cast<double>(step) * f);
        if (out) {
            Run<T, V>* yr = reinterpret_cast<Run<T, V>*>(out + row * out_row);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int i = t + nt * j;
                Run<T, V> v;
#pragma unroll
                for (int e = 0; e < V; ++e)
                    v.e[e] = static_cast<T>(static_cast<float>(static_cast<double>(u[V * j + e]) * f));
                if (i < runs) yr[i] = v;
            }
        }
    }
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Rows of `width` bytes, `step` apart (0 where there is one).
struct Rows {
    uintptr_t at;
    int64_t rows, width, step;
    __int128 end() const { return static_cast<__int128>(at) + static_cast<__int128>(rows - 1) * step + width; }
    bool same(const Rows& o) const { return at == o.at && step == o.step; }
};
Rows rows_of(const void* p, int64_t rows, int64_t row, int64_t k, int64_t size) {
    return {reinterpret_cast<uintptr_t>(p), p ? rows : 0, k * size, rows > 1 ? row * size : 0};
}
// Whether no byte is in both. Rows as far apart as the other's may lie between them;
// otherwise what counts is from where to where they reach.
bool apart(const Rows& a, const Rows& b) {
    if (a.rows == 0 || b.rows == 0 || a.end() <= b.at || b.end() <= a.at) return true;
    if (a.step != b.step || a.step == 0) return false;
    if (b.at < a.at) return apart(b, a);
    // row i of a and row j of b: b's place less a's is d + (j - i) step
    const int64_t d = static_cast<int64_t>(b.at - a.at), n = d / a.step;
    return d - n * a.step >= a.width && (n + 1 >= a.rows || d - (n + 1) * a.step <= -b.width);
}
// What the header says of each output: hidden and out may be x or the residual, and
// nothing else may be in two places.
bool outputs_apart(const rocknpu_norm_args& a, int64_t size, int64_t weight_size) {
    const Rows in[2] = {rows_of(a.x, a.rows, a.x_row, a.k, size), rows_of(a.residual, a.rows, a.residual_row, a.k, size)};
    const Rows weight = rows_of(a.weight, 1, 0, a.k, weight_size);
    const Rows to[4] = {rows_of(a.hidden, a.rows, a.hidden_row, a.k, size), rows_of(a.out, a.rows, a.out_row, a.k, size),
                        rows_of(a.a8, a.rows, a.k_pad, a.k_pad, 1), rows_of(a.scales, 1, 0, a.rows, 4)};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < i; ++j)
            if (!apart(to[i], to[j])) return false;
        for (const Rows& from : in)
            if (!(i < 2 && to[i].same(from)) && !apart(to[i], from)) return false;
        if (!apart(to[i], weight)) return false;
    }
    return true;
}

template <typename T, typename W, int V, int R>
int launch(const rocknpu_norm_args& a, int nt, hipStream_t stream) {
    constexpr int64_t kRowsOnce = 1 << 21;  // a launch holds less than 2^32 threads, a row up to 1024
    for (int64_t row = 0; row < a.rows; row += kRowsOnce) {
        const auto from = [row](auto* p, int64_t ld) { return p ? p + row * ld : p; };
        norm_a8_kernel<T, W, V, R><<<dim3(static_cast<unsigned>(std::min(a.rows - row, kRowsOnce))), dim3(nt), 0, stream>>>(
            from(static_cast<const T*>(a.x), a.x_row), from(static_cast<const T*>(a.residual), a.residual_row),
            static_cast<const W*>(a.weight), a.x_row, a.residual_row, static_cast<int>(a.k), nt,
            from(static_cast<T*>(a.hidden), a.hidden_row), a.hidden_row, from(static_cast<T*>(a.out), a.out_row), a.out_row,
            from(a.a8, a.k_pad), a.k_pad, from(a.scales, 1), a.eps);
        if (hipGetLastError() != hipSuccess) return kStatusExec;
    }
    return kStatusOk;
}

// Threads a row: two runs each (one for at most 512 rows), in whole waves, at
// most 1024. us by one run and by two, of 64, 512, 1024 and 2048 rows: 1024 f32 3.2 and
// 3.3, 3.7 and 3.9, 4.4 and 4.4, 5.7 and 5.6; 2048 f32 3.5 and 3.5, 4.5 and 4.4, 5.9 and 5.9, 11.6
// and 10.5; 4096 f32 4.2 and 3.9, 6.2 and 5.9, 12.8 and 10.6, 20.2 and 17.8; 2048 bf16 3.3 and
// 3.9, 4.0 and 4.7, 5.0 and 5.1, 6.9 and 7.4; 8192 bf16 4.4 and 4.7, 7.2 and 7.8, 14.2 and 12.9, 21.7 and 20.7.
template <typename T, typename W>
int route(const rocknpu_norm_args& a, hipStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = a.k % V == 0 && a.x_row % V == 0 && a.residual_row % V == 0 && a.hidden_row % V == 0 &&
                     a.out_row % V == 0 && a.k_pad % 8 == 0 && aligned(a.x, 16) && aligned(a.residual, 16) &&
                     aligned(a.hidden, 16) && aligned(a.out, 16) && aligned(a.weight, 16) && aligned(a.a8, 8);
    const auto threads = [&](int64_t runs, int64_t per) {
        return static_cast<int>(std::min<int64_t>(1024, ((runs + per - 1) / per + 63) / 64 * 64));
    };
    if (vec) {
        const int64_t runs = a.k / V;
        const int nt = threads(runs, a.rows <= 512 ? 1 : 2);
        const int64_t r = (runs + nt - 1) / nt;
        if (r <= 1) return launch<T, W, V, 1>(a, nt, stream);
        if (r <= 2) return launch<T, W, V, 2>(a, nt, stream);
        if (r <= 4) return launch<T, W, V, 4>(a, nt, stream);
        if (r <= 8) return launch<T, W, V, 8>(a, nt, stream);
        if constexpr (V == 4) return launch<T, W, V, 16>(a, nt, stream);
    }
    const int nt = threads(a.k, 4);
    const int64_t r = (a.k + nt - 1) / nt;
    if (r <= 4) return launch<T, W, 1, 4>(a, nt, stream);
    if (r <= 16) return launch<T, W, 1, 16>(a, nt, stream);
    return launch<T, W, 1, 64>(a, nt, stream);
}

}  // namespace
}  // namespace rk

extern "C" int rocknpu_hip_norm_a8(const rocknpu_norm_args* args, void* stream) {
    using namespace rk;
    if (!args) return kStatusInvalid;
    const rocknpu_norm_args& a = *args;
    if (a.type > ROCKNPU_TYPE_BF16 || (a.weight_type != ROCKNPU_TYPE_F32 && a.weight_type != a.type)) return kStatusInvalid;
    if (a.rows < 0 || a.rows > INT_MAX || a.k < 1 || a.k > ROCKNPU_NORM_MAX_K || a.k_pad < a.k || a.k_pad > INT_MAX)
        return kStatusInvalid;
    if (!(a.eps >= 1e-30f) || !(a.eps <= 3.402823466e38f) || !a.weight || (a.hidden && !a.residual)) return kStatusInvalid;
    const uintptr_t size = a.type == ROCKNPU_TYPE_F32 ? 4 : 2, wsize = a.weight_type == ROCKNPU_TYPE_F32 ? 4 : 2;
    if (!aligned(a.x, size) || !aligned(a.residual, size) || !aligned(a.hidden, size) || !aligned(a.out, size) ||
        !aligned(a.weight, wsize) || !aligned(a.scales, 4))
        return kStatusInvalid;
    if (a.x_row < 0 || a.residual_row < 0 || a.hidden_row < 0 || a.out_row < 0) return kStatusInvalid;
    if (a.rows > 1 && ((a.hidden && a.hidden_row < a.k) || (a.out && a.out_row < a.k))) return kStatusInvalid;
    if (a.rows == 0) return kStatusOk;
    if (!a.x || !a.a8 || !a.scales || !outputs_apart(a, static_cast<int64_t>(size), static_cast<int64_t>(wsize))) return kStatusInvalid;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.type == ROCKNPU_TYPE_F32) return route<float, float>(a, s);
    if (a.weight_type == ROCKNPU_TYPE_F32)
        return a.type == ROCKNPU_TYPE_F16 ? route<_Float16, float>(a, s) : route<__bf16, float>(a, s);
    return a.type == ROCKNPU_TYPE_F16 ? route<_Float16, _Float16>(a, s) : route<__bf16, __bf16>(a, s);
}
