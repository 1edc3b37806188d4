// Routing of tokens to experts (include/rocknpu_moe.h): the choice, and the plan
// of the experts' products.
//
// The ranking is in 64 bits: scores that differ by less than an f32's last place
// are common among hundreds of experts, and ids have to be the same whoever
// computes them.
#include "moe.h"

#include <algorithm>
#include <climits>

namespace rk {
namespace {

constexpr double kNone = -__builtin_inf();

__device__ __forceinline__ double shfl_xor(double v, int o) { return __shfl_xor(v, o, 64); }

struct RouteParams {
    const void* logits;
    const float* bias;
    int32_t* ids;
    float* weights;
    int64_t logits_row;
    int tokens, experts, top_k, groups, top_groups, group_top;
    float factor;
};

// One wave a token, lane l holding experts l, l + 64, ..; the ranks of a token's
// groups go through LDS.
template <typename T, int P, bool SIGMOID, bool NORMALISE>
__global__ __launch_bounds__(256) void route_kernel(const RouteParams p) {
    extern __shared__ double smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = blockIdx.x * 4 + wave;
    if (token >= p.tokens) return;  // a whole wave; no barrier follows
    const T* x = static_cast<const T*>(p.logits) + token * p.logits_row;
    float l[P];
    bool odd = false;
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int e = lane + 64 * j;
        l[j] = e < p.experts ? static_cast<float>(x[e]) : -__builtin_inff();
        odd |= !(l[j] < __builtin_inff());
    }
    const bool bad = __any(odd);
    double score[P], rank[P];
    double total = 0.0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        if (bad) l[j] = lane + 64 * j < p.experts ? 0.0f : -__builtin_inff();
        top = fmaxf(top, l[j]);
    }
    if constexpr (!SIGMOID) {
        top = wave_max(top);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            score[j] = l[j] == -__builtin_inff() ? 0.0 : exp(static_cast<double>(l[j]) - static_cast<double>(top));
            total += score[j];
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) total += shfl_xor(total, o);
        total = fmax(total, 1e-300);
#pragma unroll
        for (int j = 0; j < P; ++j) score[j] /= total;
    } else {
#pragma unroll
        for (int j = 0; j < P; ++j) score[j] = 1.0 / (1.0 + exp(-static_cast<double>(l[j])));
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int e = lane + 64 * j;
        rank[j] = static_cast<double>(l[j]);
        if (p.bias && !bad && l[j] != -__builtin_inff()) {
            rank[j] = score[j] + static_cast<double>(p.bias[e]);
            if (rank[j] != rank[j]) rank[j] = kNone;
        }
    }
    if (p.groups > 1) {
        double* all = smem + wave * p.experts;
        const int size = p.experts / p.groups;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e = lane + 64 * j;
            const bool scores = p.group_top == 2 && !p.bias && !bad && l[j] != -__builtin_inff();
            if (e < p.experts) all[e] = scores ? score[j] : rank[j];
        }
        // lane g: its group's best and second best; then the groups before it
        double a = kNone, b = kNone;
        if (lane < p.groups)
            for (int i = 0; i < size; ++i) {
                const double v = all[lane * size + i];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
        const double mine = p.group_top == 1 ? a : b == kNone ? kNone : a + b;
        int before = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double v = __shfl(mine, g, 64);
            before += v > mine || (v == mine && g < lane);
        }
        const uint64_t open = __ballot(lane < p.groups && before < p.top_groups);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e = lane + 64 * j;
            if (!(open >> (min(e, p.experts - 1) / size) & 1)) rank[j] = kNone;
        }
    }
    // top_k times the best that is left; lane i keeps choice i
    int id = -1;
    double chosen = 0.0;
    for (int i = 0; i < p.top_k; ++i) {
        double v = kNone, s = 0.0;
        int at = INT_MAX;
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (rank[j] > v) {
                v = rank[j];
                s = score[j];
                at = lane + 64 * j;
            }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double ov = shfl_xor(v, o), os = shfl_xor(s, o);
            const int oa = __shfl_xor(at, o, 64);
            if (ov > v || (ov == v && oa < at)) {
                v = ov;
                s = os;
                at = oa;
            }
        }
        if (at == INT_MAX) break;  // nothing is left
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (lane + 64 * j == at) rank[j] = kNone;
        if (lane == i) {
            id = at;
            chosen = s;
        }
    }
    if constexpr (NORMALISE) {
        double sum = chosen;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += shfl_xor(sum, o);
        chosen /= sum + 1e-20;
    }
    if (lane < p.top_k) {
        const int64_t at = static_cast<int64_t>(token) * p.top_k + lane;
        p.ids[at] = id;
        p.weights[at] = id < 0 ? 0.0f : bad ? __builtin_nanf("") : static_cast<float>(chosen * static_cast<double>(p.factor));
    }
}

// Lane l gets the sum over lanes 0 .. l.
__device__ __forceinline__ int scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 to rows 2 and 3
    return x;
}

// Exclusive sums over the workgroup's threads; `sums` holds 17 ints.
__device__ __forceinline__ int scan_threads(int x, int* sums, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int in = scan(x);
    if (lane == 63) sums[wave] = in;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kMoeCountThreads / 64; ++w) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    total = all;
    __syncthreads();
    return before + in - x;
}

// A block's choices by expert.
__global__ __launch_bounds__(kMoeCountThreads) void count_kernel(const int32_t* __restrict__ ids, int rows, int experts,
                                                                 int block, int32_t* __restrict__ counts) {
    __shared__ int hist[ROCKNPU_MOE_MAX_EXPERTS];
    for (int e = threadIdx.x; e < experts; e += kMoeCountThreads) hist[e] = 0;
    __syncthreads();
    const int first = blockIdx.x * block, last = min(rows - first, block) + first;
    for (int i = first + threadIdx.x; i < last; i += kMoeCountThreads) {
        const int e = ids[i];
        if (e >= 0 && e < experts) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kMoeCountThreads) counts[blockIdx.x * experts + e] = hist[e];
}

// Places a block's choices, in order: wave w takes the w-th run of the block.
// hist[w][e] counts the wave's choices of e, then holds where its next one goes.
__global__ __launch_bounds__(kMoeCountThreads) void place_kernel(const int32_t* __restrict__ ids, const MoePlan p) {
    constexpr int W = kMoeCountThreads / 64;
    extern __shared__ int hist[];
    __shared__ int sums[W + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = p.experts;
    for (int i = threadIdx.x; i < W * E; i += kMoeCountThreads) hist[i] = 0;
    __syncthreads();
    const int run = p.block / W, first = blockIdx.x * p.block + wave * run, last = min(first + run, p.rows);
    for (int i = first + lane; i < last; i += 64) {
        const int e = ids[i];
        if (e >= 0 && e < E) atomicAdd(&hist[wave * E + e], 1);
    }
    __syncthreads();
    // thread e: choices of expert e in all blocks, and in the blocks and waves before
    const int e0 = threadIdx.x;
    int all = 0, before = 0;
    if (e0 < E) {
        if (p.blocks > 1) {
            for (int b = 0; b < p.blocks; ++b) {
                const int c = p.counts[b * E + e0];
                all += c;
                before += b < static_cast<int>(blockIdx.x) ? c : 0;
            }
        } else {
            for (int w = 0; w < W; ++w) all += hist[w * E + e0];
        }
    }
    int total;
    const int offset = scan_threads(all, sums, total);
    if (e0 < E) {
        int at = offset + before;
        for (int w = 0; w < W; ++w) {
            const int c = hist[w * E + e0];
            hist[w * E + e0] = at;
            at += c;
        }
    }
    if (blockIdx.x == 0) {
        if (e0 < E) p.offsets[e0] = offset;
        if (e0 == 0) p.offsets[E] = total;
        const int n = (all + p.tile_rows - 1) / p.tile_rows;
        int tiles;
        const int t0 = scan_threads(n, sums, tiles);
        for (int t = 0; t < n; ++t) {
            p.tiles[2 * (t0 + t)] = e0;
            p.tiles[2 * (t0 + t) + 1] = offset + t * p.tile_rows;
        }
        if (e0 == 0) *p.tile_count = tiles;
    }
    __syncthreads();
    for (int i0 = first; i0 < last; i0 += 64) {
        const int i = i0 + lane;
        const int e = i < last ? ids[i] : -1;
        const bool valid = e >= 0 && e < E;
        // the lanes with the same expert
        uint64_t same = __ballot(valid);
        for (int b = 1; b < E; b <<= 1) {
            const uint64_t set = __ballot(e & b);
            same &= e & b ? set : ~set;
        }
        const int ahead = __popcll(same & ((uint64_t{1} << lane) - 1));
        int at = -1;
        if (valid) at = hist[wave * E + e] + ahead;
        __builtin_amdgcn_wave_barrier();
        if (valid && ahead == 0) hist[wave * E + e] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (valid) p.order[at] = i;
        if (i < last) p.place[i] = at;
    }
    for (int i = total + blockIdx.x * kMoeCountThreads + threadIdx.x; i < p.rows; i += gridDim.x * kMoeCountThreads)
        p.order[i] = -1;
}

template <typename T, int P>
int launch_route(const RouteParams& p, bool sigmoid, bool normalise, hipStream_t stream) {
    const dim3 grid((p.tokens + 3) / 4), block(256);
    const size_t lds = p.groups > 1 ? static_cast<size_t>(4) * p.experts * sizeof(double) : 0;
    if (sigmoid && normalise) route_kernel<T, P, true, true><<<grid, block, lds, stream>>>(p);
    else if (sigmoid) route_kernel<T, P, true, false><<<grid, block, lds, stream>>>(p);
    else if (normalise) route_kernel<T, P, false, true><<<grid, block, lds, stream>>>(p);
    else route_kernel<T, P, false, false><<<grid, block, lds, stream>>>(p);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <typename T>
int route(const RouteParams& p, bool sigmoid, bool normalise, hipStream_t stream) {
    if (p.experts <= 64) return launch_route<T, 1>(p, sigmoid, normalise, stream);
    if (p.experts <= 128) return launch_route<T, 2>(p, sigmoid, normalise, stream);
    if (p.experts <= 256) return launch_route<T, 4>(p, sigmoid, normalise, stream);
    if (p.experts <= 512) return launch_route<T, 8>(p, sigmoid, normalise, stream);
    return launch_route<T, 16>(p, sigmoid, normalise, stream);
}

int launch_plan(const int32_t* ids, const MoePlan& p, hipStream_t stream) {
    const dim3 grid(std::max(p.blocks, 1)), block(kMoeCountThreads);
    if (p.blocks > 1) {
        count_kernel<<<grid, block, 0, stream>>>(ids, p.rows, p.experts, p.block, p.counts);
        if (hipGetLastError() != hipSuccess) return kStatusExec;
    }
    const size_t lds = static_cast<size_t>(kMoeCountThreads / 64) * p.experts * sizeof(int);
    place_kernel<<<grid, block, lds, stream>>>(ids, p);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

bool moe_size_ok(int64_t tokens, int32_t experts, int32_t top_k) {
    return tokens >= 0 && experts >= 1 && experts <= ROCKNPU_MOE_MAX_EXPERTS && top_k >= 1 &&
           top_k <= ROCKNPU_MOE_MAX_TOP_K && top_k <= experts && tokens <= ROCKNPU_MOE_MAX_ROWS / top_k;
}

}  // namespace rk

extern "C" int rocknpu_hip_moe_plan_words(int64_t tokens, int32_t experts, int32_t top_k, size_t* words) {
    using namespace rk;
    if (!words || !moe_size_ok(tokens, experts, top_k)) return kStatusInvalid;
    moe_plan(tokens, experts, top_k, nullptr, words);
    return kStatusOk;
}

extern "C" int rocknpu_hip_moe_route(const rocknpu_moe_route_args* args, void* stream) {
    using namespace rk;
    if (!args) return kStatusInvalid;
    const rocknpu_moe_route_args& a = *args;
    if (!moe_size_ok(a.tokens, a.experts, a.top_k) || a.type > ROCKNPU_TYPE_BF16 || !a.plan || !aligned(a.plan, 4))
        return kStatusInvalid;
    if (a.groups < 1 || a.groups > ROCKNPU_MOE_MAX_GROUPS || a.experts % a.groups != 0 || a.top_groups < 1 ||
        a.top_groups > a.groups || a.top_groups * (a.experts / a.groups) < a.top_k)
        return kStatusInvalid;
    if (a.group_top < 1 || a.group_top > 2 || a.group_top > a.experts / a.groups) return kStatusInvalid;
    if ((a.score != ROCKNPU_MOE_SOFTMAX && a.score != ROCKNPU_MOE_SIGMOID) || !(a.factor - a.factor == 0.0f))
        return kStatusInvalid;
    const uintptr_t size = a.type == ROCKNPU_TYPE_F32 ? 4 : 2;
    if (!aligned(a.logits, size) || !aligned(a.bias, 4) || !aligned(a.ids, 4) || !aligned(a.weights, 4) || a.logits_row < 0)
        return kStatusInvalid;
    if (a.tokens > 0 && (!a.logits || !a.ids || !a.weights)) return kStatusInvalid;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.tokens > 0) {
        const RouteParams p{a.logits, a.bias, a.ids, a.weights, a.logits_row, static_cast<int>(a.tokens), a.experts, a.top_k,
                            a.groups, a.top_groups, a.group_top, a.factor};
        const bool sigmoid = a.score == ROCKNPU_MOE_SIGMOID, norm = a.normalise != 0;
        const int st = a.type == ROCKNPU_TYPE_F32   ? route<float>(p, sigmoid, norm, s)
                       : a.type == ROCKNPU_TYPE_F16 ? route<_Float16>(p, sigmoid, norm, s)
                                                    : route<__bf16>(p, sigmoid, norm, s);
        if (st != kStatusOk) return st;
    }
    return launch_plan(a.ids, moe_plan(a.tokens, a.experts, a.top_k, a.plan, nullptr), s);
}
