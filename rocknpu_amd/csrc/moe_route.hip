// Routing of tokens to experts (include/rocknpu_moe.h): the choice, and the plan
// of the experts' products.
//
// The ranking is in 64 bits: scores that differ by less than an f32's last place
// are common among hundreds of experts, and ids have to be the same whoever
// computes them. That is route_token, a wave a token. Most tokens need none of it:
// route_rows ranks by 24-bit whole numbers, 16 lanes a token, notices every token
// whose choice its rounding could have turned, and hands those to route_token.
//
// 16384 tokens over 256 experts in groups: 17.7 us (by route_token alone 65) and 7 to
// place the choices; 4096 over 64: 7.1 and 7 (17 alone); one token 5.8 to 7.9 with its
// plan. Bound by issue and latency, four waves a SIMD of which each chooses for four
// tokens; the bytes would take 4 us. A lane's 8 largest keys are sorted first (108
// operations for 16 keys) and then handed out: 24 us where every choice took the
// largest of all 16 and cleared it.
#include "moe.h"

#include <algorithm>
#include <climits>

namespace rk {
namespace {

constexpr double kNone = -__builtin_inf();

// The same 16 lanes get the result of these.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, dpp<0xB1>(v));   // lanes 1 0 3 2
    v = max(v, dpp<0x4E>(v));   // lanes 2 3 0 1
    v = max(v, dpp<0x141>(v));  // mirrored within 8
    return max(v, dpp<0x140>(v));
}
__device__ __forceinline__ float dpp_max(float v, uint32_t o) { return fmaxf(v, __uint_as_float(o)); }
__device__ __forceinline__ float row_max(float v) {
    v = dpp_max(v, dpp<0xB1>(__float_as_uint(v)));
    v = dpp_max(v, dpp<0x4E>(__float_as_uint(v)));
    v = dpp_max(v, dpp<0x141>(__float_as_uint(v)));
    return dpp_max(v, dpp<0x140>(__float_as_uint(v)));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __uint_as_float(dpp<0xB1>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x4E>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
    return v + __uint_as_float(dpp<0x140>(__float_as_uint(v)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t b = __double_as_longlong(v);
    return __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(dpp<CTRL>(static_cast<uint32_t>(b >> 32))) << 32 |
                                                     dpp<CTRL>(static_cast<uint32_t>(b))));
}
__device__ __forceinline__ double row_sum(double v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}
// How many of the row's other lanes hold more.
template <int R>
__device__ __forceinline__ void count_above(uint32_t v, int& n) {
    n += dpp<0x120 + R>(v) > v;  // row_ror
    if constexpr (R < 15) count_above<R + 1>(v, n);
}

__device__ __forceinline__ double read_lane(double v, int lane) {
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
    return __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}
// Every lane gets the wave's.
__device__ __forceinline__ double wave_max(double v) {
    v = fmax(v, dpp<0xB1>(v));
    v = fmax(v, dpp<0x4E>(v));
    v = fmax(v, dpp<0x141>(v));
    v = fmax(v, dpp<0x140>(v));
    return fmax(fmax(read_lane(v, 0), read_lane(v, 16)), fmax(read_lane(v, 32), read_lane(v, 48)));
}
__device__ __forceinline__ double wave_sum(double v) {
    v = row_sum(v);
    return (read_lane(v, 0) + read_lane(v, 16)) + (read_lane(v, 32) + read_lane(v, 48));
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct RouteParams {
    const void* logits;
    const float* bias;
    int32_t* ids;
    float* weights;
    int64_t logits_row;
    int tokens, experts, top_k, groups, top_groups, group_top;
    int normalise;
    float factor;
};

// One token by one wave, lane l holding experts l, l + 64, ..; `all` are `experts`
// doubles of the wave's own in LDS, used with groups. Lane i returns choice i.
template <typename T, int P, bool SIGMOID>
__device__ __forceinline__ int route_token(const RouteParams& p, int token, double* all) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // or what depends on it would be worked out ahead of tokens that need none of this
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
        total = fmax(wave_sum(total), 1e-300);
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
#pragma unroll 8
            for (int i = 0; i < size; ++i) {
                const double v = all[lane * size + i];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
        const double mine = p.group_top == 1 ? a : b == kNone ? kNone : a + b;
        int before = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double v = read_lane(mine, g);
            before += v > mine || (v == mine && g < lane);
        }
        const uint64_t open = __ballot(lane < p.groups && before < p.top_groups);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e = lane + 64 * j;
            if (!(open >> (min(e, p.experts - 1) / size) & 1)) rank[j] = kNone;
        }
    }
    // top_k times the best that is left, the first of equals; lane i keeps choice i
    int id = -1;
    double chosen = 0.0;
    for (int i = 0; i < p.top_k; ++i) {
        double v = rank[0];
#pragma unroll
        for (int j = 1; j < P; ++j) v = fmax(v, rank[j]);
        v = wave_max(v);
        if (v == kNone) break;  // nothing is left
        int at = -1;
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint64_t holds = __ballot(rank[j] == v);
            if (at < 0 && holds) {
                const int from = __builtin_ctzll(holds);
                at = from + 64 * j;
                s = read_lane(score[j], from);
                if (lane == from) rank[j] = kNone;
            }
        }
        if (lane == i) {
            id = at;
            chosen = s;
        }
    }
    if (p.normalise) {
        chosen /= wave_sum(chosen) + 1e-20;
    }
    if (lane < p.top_k) {
        const int64_t at = static_cast<int64_t>(token) * p.top_k + lane;
        p.ids[at] = id;
        p.weights[at] = id < 0 ? 0.0f : bad ? __builtin_nanf("") : static_cast<float>(chosen * static_cast<double>(p.factor));
    }
    return lane < p.top_k ? id : -1;
}

template <typename T, int P, bool SIGMOID>
__global__ __launch_bounds__(256) void route_token_kernel(const RouteParams p) {
    extern __shared__ double smem[];
    const int wave = threadIdx.x >> 6;
    for (int64_t token = blockIdx.x * 4 + wave; token < p.tokens; token += gridDim.x * 4)
        route_token<T, P, SIGMOID>(p, static_cast<int>(token), smem + wave * p.experts);
}

__device__ __forceinline__ void in_order(uint32_t& a, uint32_t& b) {
    const uint32_t m = min(a, b);
    a = max(a, b);
    b = m;
}
// The largest kFirst of a lane's keys (all of fewer), the largest first: sorted halves
// of 8 (Batcher's odd-even merges), of which the larger of each pair from opposite
// ends are the 8 largest, rising then falling, and a merge of those.
constexpr int kFirst = 8;
template <int N>
__device__ __forceinline__ void sort8(uint32_t* k) {
    if constexpr (N >= 2) {
        in_order(k[0], k[1]);
        if constexpr (N >= 4) in_order(k[2], k[3]);
        if constexpr (N >= 8) { in_order(k[4], k[5]); in_order(k[6], k[7]); }
    }
    if constexpr (N >= 4) {
        in_order(k[0], k[2]); in_order(k[1], k[3]);
        if constexpr (N >= 8) { in_order(k[4], k[6]); in_order(k[5], k[7]); }
        in_order(k[1], k[2]);
        if constexpr (N >= 8) in_order(k[5], k[6]);
    }
    if constexpr (N >= 8) {
        in_order(k[0], k[4]); in_order(k[1], k[5]); in_order(k[2], k[6]); in_order(k[3], k[7]);
        in_order(k[2], k[4]); in_order(k[3], k[5]);
        in_order(k[1], k[2]); in_order(k[3], k[4]); in_order(k[5], k[6]);
    }
}
template <int P, int F>
__device__ __forceinline__ void first_keys(uint32_t (&key)[P], uint32_t (&f)[F]) {
    if constexpr (P <= 8) {
        sort8<P>(key);
#pragma unroll
        for (int j = 0; j < F; ++j) f[j] = key[j];
    } else {
        sort8<8>(key);
        sort8<8>(key + 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = max(key[j], key[15 - j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) in_order(f[j], f[j + 4]);
#pragma unroll
        for (int j = 0; j < 8; j += 4) { in_order(f[j], f[j + 2]); in_order(f[j + 1], f[j + 3]); }
#pragma unroll
        for (int j = 0; j < 8; j += 2) in_order(f[j], f[j + 1]);
    }
}

// All ones, or for a logit of -inf zero (no branch around what it masks).
__device__ __forceinline__ uint32_t open_mask(float logit) { return logit == -__builtin_inff() ? 0u : ~0u; }

constexpr int kRowsTopK = 16;      // choices that route_rows holds, one a lane
constexpr int kRowsExperts = 256;  // experts, 16 a lane and 8 bits of a key
constexpr float kUnit = 0x1p20f;   // units of a key's value

// What of a routing's plan a block of tokens works out along with its choices.
struct RouteBlocks {
    MoePlan plan;
    int tokens;  // of a block
    int size;    // experts of a group
    int shift;   // a group's lanes are 1 << shift
    int vec;     // logits and bias can be loaded 16 bytes at a time
};

__device__ void place_block(const int32_t* ids, int first, int last, int run, const MoePlan& p, int* hist, int* sums, int all,
                            int before, bool leads);

// A block of tokens by 16 lanes each, lane l of them holding P neighbouring experts
// of a group. An expert's key has its rank in the upper 24 bits and 255 - its
// index in the lower 8, so a maximum is the best and, of equals, the first; 0 is an
// expert that cannot be chosen. Ranks are
//   - without a bias, 16-bit logits: their bits, in order: exact;
//   - without a bias, f32 logits: 2^20 (logit - the token's largest), from -16 up;
//   - with a bias: 2^20 (score + bias), within +-7.9.
// The last two are truncated from f32 values that are within 0.6 of a unit of the
// 64-bit one: 0.25 for the last place of a sum with the bias (0.5 for that of a
// logit's distance from the largest), 0.13 for the reciprocal or the exponential and 0.1
// for the roundings around it (and a softmax's sum of up to 256 within 1.3 units of its share, the
// same for all). Keys that differ by four units or more are in the right order,
// and sums of two that differ by eight. Where two choices, or the last one and the best that is left,
// differ by less, or the last open group and the best closed one, or where a
// value does not fit, the token goes to route_token. The weights are worked out
// in 64 bits from the chosen logits.
template <typename T, int P, bool SIGMOID>
__global__ __launch_bounds__(1024) void route_rows_kernel(const RouteParams p, const RouteBlocks b) {
    extern __shared__ double smem[];
    __shared__ int32_t chosen_ids[64 * kRowsTopK];
    __shared__ int hist[16 * kRowsExperts];
    __shared__ int sums[17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int l16 = lane & 15;
    const bool alone = b.plan.blocks == 1;
    double* all = smem + wave * p.experts;
    for (int i = threadIdx.x; i < (alone ? waves : 1) * p.experts; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    const int size = b.size, group = l16 >> b.shift, at0 = (l16 & ((1 << b.shift) - 1)) * P;
    const int base = blockIdx.x * b.tokens, end = min(base + b.tokens, p.tokens);
    const bool exact = sizeof(T) == 2 && !p.bias;
    for (int t0 = base + wave * 4; t0 < end; t0 += 4 * waves) {
        const int token = t0 + (lane >> 4);
        const bool active = token < end;
        const T* x = static_cast<const T*>(p.logits) + min(token, end - 1) * p.logits_row;
        int e0 = group * size + at0;
        asm volatile("" : "+v"(e0));  // or 16 addresses would be kept over the passes, in memory
        float l[P];
        bool odd = false;  // the token goes to route_token
        if (b.vec) {
            constexpr int V = P * sizeof(T) >= 16 ? 16 / sizeof(T) : P;
            struct alignas(V * sizeof(T)) Run {
                T e[V];
            };
#pragma unroll
            for (int j = 0; j < P; j += V) {
                Run r = {};
                if (group < p.groups && at0 + j < size) r = *reinterpret_cast<const Run*>(x + e0 + j);
#pragma unroll
                for (int i = 0; i < V; ++i) l[j + i] = static_cast<float>(r.e[i]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j) l[j] = group < p.groups && at0 + j < size ? static_cast<float>(x[e0 + j]) : 0.0f;
        }
        float bias[P];  // asked for together with the logits
        if (p.bias) {
            constexpr int V = P < 4 ? P : 4;
            struct alignas(V * 4) Run {
                float e[V];
            };
            if (b.vec) {
#pragma unroll
                for (int j = 0; j < P; j += V) {
                    const Run r = *reinterpret_cast<const Run*>(p.bias + min(e0 + j, p.experts - V));
#pragma unroll
                    for (int i = 0; i < V; ++i) bias[j + i] = r.e[i];
                }
            } else {
#pragma unroll
                for (int j = 0; j < P; ++j) bias[j] = p.bias[min(e0 + j, p.experts - 1)];
            }
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < P; ++j) {
            odd |= !(l[j] < __builtin_inff());
            if (!(group < p.groups && at0 + j < size)) l[j] = -__builtin_inff();
            top = fmaxf(top, l[j]);
        }
        top = row_max(top);
        uint32_t key[P];
        if (exact) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const T h = static_cast<T>(l[j] + 0.0f);  // -0 as 0
                uint16_t u;
                __builtin_memcpy(&u, &h, 2);
                const uint32_t o = u & 0x8000 ? u ^ 0xFFFFu : u | 0x8000u;
                key[j] = open_mask(l[j]) & (o << 16 | (255 - (e0 + j)));
            }
        } else {
            float y[P];
            float floor = -8.0f;
            if (!p.bias) {
                floor = -16.0f;
#pragma unroll
                for (int j = 0; j < P; ++j) y[j] = l[j] - top;
            } else {
                float scale = 1.0f;
                if constexpr (SIGMOID) {
#pragma unroll
                    for (int j = 0; j < P; ++j)
                        y[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -1.44269504f));
                } else {
                    float total = 0.0f;
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        y[j] = __builtin_amdgcn_exp2f((l[j] - top) * 1.44269504f);
                        total += l[j] == -__builtin_inff() ? 0.0f : y[j];
                    }
                    scale = __builtin_amdgcn_rcpf(row_sum(total));
                }
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const bool real = l[j] != -__builtin_inff();
                    y[j] = y[j] * scale + bias[j];
                    odd |= real && !(fabsf(y[j]) < 7.9f);
                }
            }
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const int q = static_cast<int>(fmaxf(y[j], floor) * kUnit) - static_cast<int>(floor * kUnit);
                key[j] = open_mask(l[j]) & (static_cast<uint32_t>(min(max(q, 1), 0xFFFFFF)) << 8 | (255 - (e0 + j)));
            }
        }
        if (p.groups > 1) {
            uint32_t a = 0, c = 0;  // the group's best and second best
#pragma unroll
            for (int j = 0; j < P; ++j) {
                c = max(c, min(a, key[j]));
                a = max(a, key[j]);
            }
            const auto join = [&](uint32_t oa, uint32_t oc) {
                c = max(min(a, oa), max(c, oc));
                a = max(a, oa);
            };
            if (b.shift >= 1) join(dpp<0xB1>(a), dpp<0xB1>(c));
            if (b.shift >= 2) join(dpp<0x4E>(a), dpp<0x4E>(c));
            if (b.shift >= 3) join(dpp<0x141>(a), dpp<0x141>(c));
            const uint32_t rank = p.group_top == 1 ? a >> 8 : c == 0 ? 0 : (a >> 8) + (c >> 8);
            int above = 0;
            count_above<1>(rank << 6 | (63 - group), above);
            const bool open = above < p.top_groups << b.shift;
            const uint32_t closed = row_max(open ? 0 : rank), least = ~row_max(open ? ~rank : 0);
            odd |= !exact && closed != 0 && least - closed < 8;
            if (!open)
#pragma unroll
                for (int j = 0; j < P; ++j) key[j] = 0;
        }
        // lane i keeps choice i, and the two that come behind the last
        const bool pairs = p.top_k <= kRowsTopK - 2 && (SIGMOID || !p.bias);
        // every lane's first keys in order: the best that is left is the largest of the
        // lanes' next
        constexpr int F = P < kFirst ? P : kFirst;
        uint32_t next[F];
        first_keys(key, next);
        int given = 0;
        uint32_t mine = 0, before = 0xFFFFFFFF;
        bool near = false;  // the choice before may be of lower rank
#pragma unroll 1
        for (int i = 0; i < p.top_k + (exact ? 0 : pairs ? 2 : 1); ++i) {
            const uint32_t best = row_max(next[0]);
            const bool close = !exact && i > 0 && best != 0 && (before >> 8) - (best >> 8) < 4, here = l16 == i;
            mine = here ? best : mine;
            near |= here && close;
            odd |= i == kRowsTopK && close;
            before = best;
            // the lane it came from moves on (by masks: a choice between neighbours in an
            // array would be made an index, and that a chain of choices)
            const uint32_t taken = next[0] == best ? ~0u : 0u;
            given += best != 0 ? taken & 1 : 0;
#pragma unroll
            for (int j = 0; j + 1 < F; ++j) next[j] = (next[j + 1] & taken) | (next[j] & ~taken);
            next[F - 1] &= ~taken;
        }
        if constexpr (P > kFirst) odd |= given >= kFirst;  // the lane may hold another
        int id = mine ? 255 - static_cast<int>(mine & 255) : -1;
        double w = 0.0;
        if (id >= 0) {
            const double v = static_cast<double>(static_cast<float>(x[id]));
            if constexpr (SIGMOID) w = 1.0 / (1.0 + exp(-v));
            else w = exp(v - static_cast<double>(top));
        }
        if (__any(near)) {
            const uint32_t behind = dpp<0x101>(static_cast<uint32_t>(near));  // of the next choice
            odd |= near && (behind || !pairs);
            // one of two near ones: they change places where their 64-bit ranks say so
            double rank = w;
            if (id >= 0) rank = p.bias ? w + static_cast<double>(p.bias[id]) : static_cast<double>(static_cast<float>(x[id]));
            // (all lanes read their neighbours' before any takes one)
            const double w_up = dpp<0x111>(w), w_down = dpp<0x101>(w), rank_up = dpp<0x111>(rank), rank_down = dpp<0x101>(rank);
            const double ow = near ? w_up : w_down, orank = near ? rank_up : rank_down;
            const int up = static_cast<int>(dpp<0x111>(static_cast<uint32_t>(id))), down = static_cast<int>(dpp<0x101>(static_cast<uint32_t>(id)));
            const int oid = near ? up : down;
            const bool wrong = near ? rank > orank || (rank == orank && id < oid) : orank > rank || (rank == orank && oid < id);
            if ((near || behind) && wrong) {
                id = oid;
                w = ow;
            }
        }
        if (l16 >= p.top_k) w = 0.0;
        if (p.normalise) {
            const double sum = row_sum(w);
            // softmax: the 1e-20 stands beside the sum over the total, which is 1 to 256
            if constexpr (!SIGMOID) odd |= id >= 0 && sum < 1e-7;
            w /= sum + 1e-20;
        } else if constexpr (!SIGMOID) {
            double total = 0.0;
#pragma unroll
            for (int j = 0; j < P; ++j)
                if (l[j] != -__builtin_inff()) total += exp(static_cast<double>(l[j]) - static_cast<double>(top));
            w /= fmax(row_sum(total), 1e-300);
        }
        const uint64_t odd_lanes = __ballot(odd);
        const auto note = [&](int t, int i, int e) {  // choice i of token t fell on e
            if (alone) chosen_ids[(t - base) * p.top_k + i] = e;
            else if (e >= 0) atomicAdd(&hist[e], 1);
        };
        if (active && l16 < p.top_k && !(odd_lanes >> (lane & 48) & 0xFFFF)) {
            const int64_t at = static_cast<int64_t>(token) * p.top_k + l16;
            p.ids[at] = id;
            p.weights[at] = id < 0 ? 0.0f : static_cast<float>(w * static_cast<double>(p.factor));
            note(token, l16, id);
        }
        for (int q = 0; q < 4; ++q)
            if ((odd_lanes >> (16 * q) & 0xFFFF) && t0 + q < end) {
                const int e = route_token<T, P >= 4 ? P / 4 : 1, SIGMOID>(p, t0 + q, all);
                if (lane < p.top_k) note(t0 + q, lane, e);
            }
    }
    __syncthreads();
    if (!alone) {
        for (int e = threadIdx.x; e < p.experts; e += blockDim.x) b.plan.counts[blockIdx.x * p.experts + e] = hist[e];
        return;
    }
    // the only block: place its choices too
    const int rows = b.plan.rows, run = (rows + 64 * waves - 1) / (64 * waves) * 64;
    place_block(chosen_ids, 0, rows, run, b.plan, hist, sums, 0, 0, true);
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

// Exclusive sums over the workgroup's threads (at most 1024); `sums` holds 16 ints.
__device__ __forceinline__ int scan_threads(int x, int* sums, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int in = scan(x);
    if (lane == 63) sums[wave] = in;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < waves; ++w) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    total = all;
    __syncthreads();
    return before + in - x;
}

// Places choices first .. last - 1 in order: wave w takes the w-th run of them (whole
// chunks of 64). hist (zeros [waves][experts]) counts a wave's choices of e, then holds
// where its next one goes. Thread e gives the choices of expert e in all blocks, and
// in those before; with one block, zeros. The workgroup that leads writes the offsets
// and the tiles. At least `experts` threads.
__device__ void place_block(const int32_t* ids, int first, int last, int run, const MoePlan& p, int* hist, int* sums, int all,
                            int before, bool leads) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, E = p.experts;
    const int from = min(first + wave * run, last), to = min(from + run, last);
    for (int i = from + lane; i < to; i += 64) {
        const int e = ids[i];
        if (e >= 0 && e < E) atomicAdd(&hist[wave * E + e], 1);
    }
    __syncthreads();
    const int e0 = threadIdx.x;
    if (e0 < E && p.blocks == 1)
        for (int w = 0; w < waves; ++w) all += hist[w * E + e0];
    int total;
    const int offset = scan_threads(all, sums, total);
    if (e0 < E) {
        int at = offset + before;
        for (int w = 0; w < waves; ++w) {
            const int c = hist[w * E + e0];
            hist[w * E + e0] = at;
            at += c;
        }
    }
    if (leads) {
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
    int bits = 0;
    while (1 << bits < E) ++bits;
    for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        const int e = i < to ? ids[i] : -1;
        const bool valid = e >= 0 && e < E;
        // the lanes with the same expert
        uint64_t same = __ballot(valid);
        for (int k = 0; k < bits; ++k) {
            const uint64_t set = __ballot(e >> k & 1);
            same &= e >> k & 1 ? set : ~set;
        }
        const int ahead = __popcll(same & ((uint64_t{1} << lane) - 1));
        int at = -1;
        if (valid) at = hist[wave * E + e] + ahead;
        __builtin_amdgcn_wave_barrier();
        if (valid && ahead == 0) hist[wave * E + e] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (valid) p.order[at] = i;
        if (i < to) p.place[i] = at;
    }
    for (int i = total + blockIdx.x * blockDim.x + threadIdx.x; i < p.rows; i += gridDim.x * blockDim.x) p.order[i] = -1;
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

// Places `each` counting blocks' choices a workgroup. 1024 / 2^shift threads an expert
// add up the blocks' counts.
__global__ __launch_bounds__(kMoeCountThreads) void place_kernel(const int32_t* __restrict__ ids, const MoePlan p, int each,
                                                                 int shift) {
    constexpr int W = kMoeCountThreads / 64;
    extern __shared__ int hist_of_waves[];
    __shared__ int sums[W], in_all[ROCKNPU_MOE_MAX_EXPERTS], in_before[ROCKNPU_MOE_MAX_EXPERTS];
    const int t = threadIdx.x, E = p.experts;
    for (int i = t; i < W * E; i += kMoeCountThreads) hist_of_waves[i] = 0;
    in_all[t] = in_before[t] = 0;
    __syncthreads();
    const int block0 = blockIdx.x * each;
    if (p.blocks > 1) {
        const int e = t & ((1 << shift) - 1), parts = kMoeCountThreads >> shift;
        if (e < E) {
            int all = 0, before = 0;
#pragma unroll 8
            for (int b = t >> shift; b < p.blocks; b += parts) {
                const int c = p.counts[b * E + e];
                all += c;
                before += b < block0 ? c : 0;
            }
            atomicAdd(&in_all[e], all);
            atomicAdd(&in_before[e], before);
        }
        __syncthreads();
    }
    const int64_t first = static_cast<int64_t>(block0) * p.block;
    const int last = static_cast<int>(min(first + static_cast<int64_t>(each) * p.block, static_cast<int64_t>(p.rows)));
    const int span = each * p.block, run = (span + 64 * W - 1) / (64 * W) * 64;
    place_block(ids, static_cast<int>(first), last, run, p, hist_of_waves, sums, in_all[t], in_before[t], blockIdx.x == 0);
}

template <typename T, int P>
int launch_tokens(const RouteParams& p, bool sigmoid, hipStream_t stream) {
    const dim3 grid(std::min((p.tokens + 3) / 4, 1 << 22)), block(256);  // a launch holds less than 2^32 threads
    const size_t lds = p.groups > 1 ? static_cast<size_t>(4) * p.experts * sizeof(double) : 0;
    if (sigmoid) route_token_kernel<T, P, true><<<grid, block, lds, stream>>>(p);
    else route_token_kernel<T, P, false><<<grid, block, lds, stream>>>(p);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <typename T, int P>
int launch_rows(const RouteParams& p, const RouteBlocks& b, bool sigmoid, hipStream_t stream) {
    // 16 waves of four tokens each; a single block takes as many waves as its tokens
    // and experts need
    const int threads = b.plan.blocks > 1 ? 1024 : std::max((p.tokens + 3) / 4 * 64, (p.experts + 63) / 64 * 64);
    const dim3 grid(b.plan.blocks), block(threads);
    const size_t lds = p.groups > 1 ? static_cast<size_t>(threads / 64) * p.experts * sizeof(double) : 0;
    if (sigmoid) route_rows_kernel<T, P, true><<<grid, block, lds, stream>>>(p, b);
    else route_rows_kernel<T, P, false><<<grid, block, lds, stream>>>(p, b);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <typename T>
int route(const RouteParams& p, const MoePlan& plan, bool sigmoid, bool* placed, bool* counted, hipStream_t stream) {
    *placed = *counted = false;
    // route_rows: groups of whole lanes, and ranks that its keys hold
    const int lanes = 16 / p.groups, size = p.experts / p.groups;
    if (p.top_k <= kRowsTopK && p.experts <= kRowsExperts && 16 % p.groups == 0 &&
        (p.groups == 1 || p.group_top == 1 || p.bias)) {
        const int each = (size + lanes - 1) / lanes;
        const int P = each <= 1 ? 1 : each <= 2 ? 2 : each <= 4 ? 4 : each <= 8 ? 8 : 16;
        const int run = std::min<int>(P * sizeof(T), 16);
        int shift = 0;
        while (1 << shift < lanes) ++shift;
        const RouteBlocks b{plan, plan.block / p.top_k, size, shift,
                            aligned(p.logits, run) && p.logits_row * sizeof(T) % run == 0 && size % (run / static_cast<int>(sizeof(T))) == 0 &&
                                size % std::min(P, 4) == 0 && aligned(p.bias, 4 * std::min(P, 4))};
        *counted = true;
        *placed = plan.blocks == 1;
        if (P == 1) return launch_rows<T, 1>(p, b, sigmoid, stream);
        if (P == 2) return launch_rows<T, 2>(p, b, sigmoid, stream);
        if (P == 4) return launch_rows<T, 4>(p, b, sigmoid, stream);
        if (P == 8) return launch_rows<T, 8>(p, b, sigmoid, stream);
        return launch_rows<T, 16>(p, b, sigmoid, stream);
    }
    if (p.experts <= 64) return launch_tokens<T, 1>(p, sigmoid, stream);
    if (p.experts <= 128) return launch_tokens<T, 2>(p, sigmoid, stream);
    if (p.experts <= 256) return launch_tokens<T, 4>(p, sigmoid, stream);
    if (p.experts <= 512) return launch_tokens<T, 8>(p, sigmoid, stream);
    return launch_tokens<T, 16>(p, sigmoid, stream);
}

int launch_plan(const int32_t* ids, const MoePlan& p, bool counted, hipStream_t stream) {
    if (p.blocks > 1 && !counted) {
        count_kernel<<<dim3(p.blocks), dim3(kMoeCountThreads), 0, stream>>>(ids, p.rows, p.experts, p.block, p.counts);
        if (hipGetLastError() != hipSuccess) return kStatusExec;
    }
    // at most 64 workgroups: every one reads all blocks' counts
    const int each = std::max((p.blocks + 63) / 64, 1);
    int shift = 0;
    while (1 << shift < p.experts) ++shift;
    const dim3 grid(std::max((p.blocks + each - 1) / each, 1));
    const size_t lds = static_cast<size_t>(kMoeCountThreads / 64) * p.experts * sizeof(int);
    place_kernel<<<grid, dim3(kMoeCountThreads), lds, stream>>>(ids, p, each, shift);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

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
    const MoePlan plan = moe_plan(a.tokens, a.experts, a.top_k, a.plan, nullptr);
    bool counted = false;
    if (a.tokens > 0) {
        const RouteParams p{a.logits, a.bias, a.ids, a.weights, a.logits_row, static_cast<int>(a.tokens), a.experts, a.top_k,
                            a.groups, a.top_groups, a.group_top, a.normalise != 0, a.factor};
        const bool sigmoid = a.score == ROCKNPU_MOE_SIGMOID;
        bool placed;
        const int st = a.type == ROCKNPU_TYPE_F32   ? route<float>(p, plan, sigmoid, &placed, &counted, s)
                       : a.type == ROCKNPU_TYPE_F16 ? route<_Float16>(p, plan, sigmoid, &placed, &counted, s)
                                                    : route<__bf16>(p, plan, sigmoid, &placed, &counted, s);
        if (st != kStatusOk || placed) return st;
    }
    return launch_plan(a.ids, plan, counted, s);
}
