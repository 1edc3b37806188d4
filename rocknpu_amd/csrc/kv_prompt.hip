// Attention of many rows over the cache: prompts, and pieces of them.
//
// A workgroup takes a tile of rows of one sequence and kv head (the step's
// tokens times the kv head's heads, so that keys and values serve all of them),
// 32 rows a wave. Two blocks at a time pass through LDS: the codes are converted
// once per workgroup, into the order in which v_mfma_f32_32x32x16 takes them,
// while the blocks before are worked on and those behind are on their way from
// memory. Scores: keys (32 tokens x 16 dims) times queries; a lane ends up with
// 16 tokens of one row, so maximum and sum are per lane but for one exchange,
// and the weights are the second operand of the next product, values (32 dims x
// 16 tokens) times weights, as they stand.
//
// Per block and wave D/16 + D/16 matrix instructions of 32 cycles, and for each
// of a lane's 16 scores a fused multiply-add, an exponential (16 cycles), half a
// maximum, conversion and sum each: matrix and vector units are both near their
// rate with 128 dims, the vector unit is what bounds 64 dims.
#include "kv_attend.h"

namespace rk {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));
typedef float float2v __attribute__((ext_vector_type(2)));

// f16 weights are held times 2^kBias, and the row's reference M follows the
// maximum only when that grows by more than kSlack: rescaling the output costs
// as much as a block's exponentials. 2^(kBias + kSlack) stays below f16's 65504.
constexpr float kBias = 9.0f, kSlack = 6.0f;
// bytes of a 512-byte run of operands in LDS, padded so that the writers' 8
// lanes a cycle meet 8 different 16-byte columns
constexpr int kKeyRun = 528, kValueRun = 544;

template <int D>
constexpr int prompt_waves() { return D <= 128 ? 8 : 4; }

template <int D>
struct StageRegs {
    static constexpr int kPieces = 2 * 2 * kKvBlock * D / 16;  // 16-byte pieces of two blocks
    static constexpr int kEach = (kPieces + 64 * prompt_waves<D>() - 1) / (64 * prompt_waves<D>());
    uint4 raw[kEach];
};

struct StageMeta {
    int page[2], start[2];
    float sk[2], sv[2];
};

template <int D>
constexpr int key_bytes() { return D / 8 * kKeyRun; }
template <int D>
constexpr int block_bytes_lds() { return key_bytes<D>() + D / 8 * kValueRun; }

// Fetches this thread's pieces of the two blocks.
template <int D>
__device__ __forceinline__ void fetch(const uint8_t* pages, const StageMeta& m, StageRegs<D>& r) {
    constexpr int kThreads = 64 * prompt_waves<D>(), kPer = 2 * kKvBlock * D / 16;
#pragma unroll
    for (int i = 0; i < StageRegs<D>::kEach; ++i) {
        const int at = threadIdx.x + i * kThreads, blk = at / kPer;
        r.raw[i] = *reinterpret_cast<const uint4*>(pages + static_cast<int64_t>(blk ? m.page[1] : m.page[0]) * (64 * D) +
                                                   at % kPer * 16);
    }
}

// Converts them into LDS. Values become bf16 for f32 calls, else f16.
template <int D, bool PAIR>
__device__ __forceinline__ void place(const StageRegs<D>& r, uint8_t* lds) {
    constexpr int kThreads = 64 * prompt_waves<D>(), kPer = 2 * kKvBlock * D / 16;
#pragma unroll
    for (int i = 0; i < StageRegs<D>::kEach; ++i) {
        const int at = threadIdx.x + i * kThreads, blk = at / kPer, piece = at % kPer;
        uint8_t* to = lds + blk * block_bytes_lds<D>();
        const uint4 w = r.raw[i];
        if (piece < kPer / 2) {  // keys: token, 16 dims
            const int step = piece / 128 * 4 + piece % 4, t = piece / 4 % 32;
            uint8_t* p = to + step * 2 * kKeyRun + t * 16;
            *reinterpret_cast<half8*>(p) = codes_to_half(w.x, w.y);
            *reinterpret_cast<half8*>(p + kKeyRun) = codes_to_half(w.z, w.w);
        } else {  // values: dims d and d + 16, 8 tokens
            const int v = piece - kPer / 2;
            uint8_t* p = to + key_bytes<D>() + (v / 64 * 4 + v % 4) * kValueRun + v / 4 % 16 * 16;
            if constexpr (PAIR) {
                *reinterpret_cast<bhalf8*>(p) = codes_to_bhalf(w.x, w.y);
                *reinterpret_cast<bhalf8*>(p + 256) = codes_to_bhalf(w.z, w.w);
            } else {
                *reinterpret_cast<half8*>(p) = codes_to_half(w.x, w.y);
                *reinterpret_cast<half8*>(p + 256) = codes_to_half(w.z, w.w);
            }
        }
    }
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

__device__ __forceinline__ float tanh_fast(float x) {
    // 1 - 2 / (1 + e^2x): its error is of 1, not of small results
    return 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + exp2_fast(2.0f * kLog2e * x));
}

template <int TYPE, int D>
__global__ __launch_bounds__(64 * prompt_waves<D>()) void kv_prompt_kernel(KvAttend p, int tiles) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    constexpr bool PAIR = TYPE == ROCKNPU_KV_F32;
    constexpr int kParts = PAIR ? 2 : 1, kWaves = prompt_waves<D>(), kTile = 32 * kWaves;
    const rocknpu_kv_cache& c = p.c;
    const rocknpu_kv_attention_args& a = p.a;
    __shared__ alignas(16) uint8_t lds[2][2 * block_bytes_lds<D>()];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the tiles with the most blocks first, a tile's kv heads side by side (one each per XCD where they are 8)
    const int h = blockIdx.x % c.kv_heads, slot_at = blockIdx.x / c.kv_heads % p.slots;
    const int tile = tiles - 1 - blockIdx.x / c.kv_heads / p.slots;
    const KvSlot mine = kv_slot(p, slot_at);
    const int b = mine.seq;
    if (b < 0) return;
    const KvSpan s = uniform(kv_span(a.past, a.cu, b, static_cast<int>(a.rows), static_cast<int>(a.max_new)));
    const int rows = s.n * p.group, r0 = tile * kTile;
    if (r0 >= rows) return;
    const int total = s.past + s.n, gone = uniform(max(c.dropped[b], 0));
    const int held = min((total + kKvBlock - 1) / kKvBlock - gone, c.max_blocks);
    const int prefix = a.prefix ? uniform(a.prefix[b]) : 0;
    const int64_t entry_row = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks;
    const KvRange range = kv_range(a, c.starts + entry_row, held, gone, s.past + r0 / p.group,
                                   s.past + (min(r0 + kTile, rows) - 1) / p.group, prefix);
    const int count = range.count();
    const int chunk = (count + mine.splits - 1) / mine.splits;
    const int begin = mine.split * chunk, end = min(begin + chunk, count);
    const int64_t slot = (static_cast<int64_t>(h) * p.row_tiles + tile) * p.slots + slot_at;
    if (begin >= end && mine.splits > 1) {
        if (tid < kTile) {
            p.part_state[(slot * kTile + tid) * 2] = -__builtin_inff();
            p.part_state[(slot * kTile + tid) * 2 + 1] = 0.0f;
        }
        return;
    }

    const int w0 = r0 + wave * 32;
    const bool active = w0 < rows;
    const int row = min(w0 + n, rows - 1), head = h * p.group + row % p.group, qpos = s.past + row / p.group;
    const int q0 = s.past + min(w0, rows - 1) / p.group, q1 = s.past + (min(w0 + 32, rows) - 1) / p.group;
    half8 q[kParts][D / 16];
    float unit;
    {
        const T* src = static_cast<const T*>(a.q) + (s.row0 + row / p.group) * a.q_row + head * a.q_head + half * 8;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            float x[8];
            load8<TYPE>(src + i * 16, p.vec_q, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        }
        const float power = row_power(fmaxf(top, other_half(top)));
        unit = a.scale / power;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            float x[8];
            load8<TYPE>(src + i * 16, p.vec_q, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[e] * power;
                q[0][i][e] = static_cast<_Float16>(v);
                if constexpr (PAIR) q[1][i][e] = static_cast<_Float16>(v - static_cast<float>(q[0][i][e]));
            }
        }
    }
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const bool plain = a.softcap == 0.0f && !a.slopes;

    float16v o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = float16v{};
    float ref = -__builtin_inff(), sum = 0.0f;

    // a stage's two blocks: the second may lie past the end, and is then masked whole (its data is the first's)
    const auto look_up = [&](int stage, StageMeta& m) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = range.entry(min(begin + 2 * stage + i, end - 1));
            m.page[i] = __builtin_amdgcn_readfirstlane(c.table[entry_row + at]);
            m.start[i] = __builtin_amdgcn_readfirstlane(c.starts[entry_row + at]);
        }
    };
    const auto look_up_scales = [&](int stage, StageMeta& m) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool ok = m.page[i] >= 0 && m.page[i] < c.n_pages;
            m.page[i] = ok ? m.page[i] : 0;
            const float2 sc = reinterpret_cast<const float2*>(c.scales)[m.page[i]];
            m.sk[i] = kv_scale(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(sc.x))), ok);
            m.sv[i] = kv_scale(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(sc.y))), ok);
            if (begin + 2 * stage + i >= end) m.start[i] = 0x7fffff00;
        }
    };
    const int stages = (end - begin + 1) / 2;
    StageMeta m0{}, m1{}, m2{};  // stages s, s + 1, s + 2
    StageRegs<D> regs;
    if (stages > 0) {
        look_up(0, m0);
        look_up(1, m1);
        look_up_scales(0, m0);
        fetch<D>(c.pages, m0, regs);
        look_up_scales(1, m1);
        place<D, PAIR>(regs, lds[0]);
        fetch<D>(c.pages, m1, regs);
        look_up(2, m2);
    }
    __syncthreads();
    for (int st = 0; st < stages; ++st) {
        const uint8_t* now = lds[st & 1];
        if (st + 1 < stages) place<D, PAIR>(regs, lds[(st + 1) & 1]);
        look_up_scales(st + 2, m2);
        if (st + 2 < stages) fetch<D>(c.pages, m2, regs);
        StageMeta m3{};
        look_up(st + 3, m3);

        // blocks that no row of the wave sees
        bool any[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            any[i] = active && m0.start[i] < total && (!a.causal || m0.start[i] <= q1 || m0.start[i] < prefix) &&
                     (a.window == 0 || m0.start[i] + kKvBlock > q0 - a.window + 1 || m0.start[i] < prefix);
        if (any[0] || any[1]) {
            float16v x[2];
            float most = -__builtin_inff(), factor[2], shift[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[i] = float16v{};
                const uint8_t* keys = now + i * block_bytes_lds<D>() + half * kKeyRun + n * 16;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const half8 key = *reinterpret_cast<const half8*>(keys + k * 2 * kKeyRun);
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        x[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, q[part][k], x[i], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // x[i][r]: token 8 (r / 4) + 4 half + r % 4
                const float lift = __log2f(m0.sv[i]);
                factor[i] = unit * m0.sk[i] * kLog2e;
                shift[i] = lift;
                if (plain && kv_all_seen(a, m0.start[i], q0, q1, prefix, total)) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) most = fmaxf(most, __builtin_fmaf(x[i][r], factor[i], lift));
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int kpos = m0.start[i] + r / 4 * 8 + half * 4 + r % 4;
                        float y;
                        if (plain) {
                            y = __builtin_fmaf(x[i][r], factor[i], lift);
                        } else {
                            y = x[i][r] * (unit * m0.sk[i]);
                            if (a.softcap != 0.0f)
                                y = a.softcap * (PAIR ? tanhf(y / a.softcap) : tanh_fast(y / a.softcap));
                            if (a.slopes) y += slope * static_cast<float>(kpos - qpos);
                            y = __builtin_fmaf(y, kLog2e, lift);
                        }
                        x[i][r] = kv_seen(a, kpos, qpos, prefix, total) ? y : -__builtin_inff();
                        most = fmaxf(most, x[i][r]);
                    }
                    factor[i] = 1.0f;
                    shift[i] = 0.0f;
                }
            }
            most = fmaxf(most, other_half(most));
            if (__any(most > ref + kSlack || (ref == -__builtin_inff() && most != ref))) {
                const float to = fmaxf(ref, most);
                const float keep = ref == to ? 1.0f : exp2_fast(ref - to);
                ref = to;
                sum *= keep;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] *= keep;
            }
            const float base = (PAIR ? 0.0f : kBias) - (ref == -__builtin_inff() ? 0.0f : ref);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float off = shift[i] + base;
                float e[16], got = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) e[r] = exp2_fast(__builtin_fmaf(x[i][r], factor[i], off));
                const uint8_t* values = now + i * block_bytes_lds<D>() + key_bytes<D>() + half * kValueRun + n * 16;
                if constexpr (PAIR) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        float ee[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            ee[j] = e[j / 4 * 8 + m * 4 + j % 4];
                            got += ee[j];
                        }
                        bhalf8 w[3];
                        split_bhalf(ee, w);
#pragma unroll
                        for (int d = 0; d < D / 32; ++d) {
                            const bhalf8 value = *reinterpret_cast<const bhalf8*>(values + (d * 4 + m * 2) * kValueRun);
#pragma unroll
                            for (int part = 0; part < 3; ++part)
                                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value, w[part], o[d], 0, 0, 0);
                        }
                    }
                } else {
                    union {
                        half2v h[4];
                        half8 v;
                    } w[2];
                    half2v least = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int r = j / 2 * 8 + m * 4 + j % 2 * 2;
                            w[m].h[j] = __builtin_convertvector(float2v{e[r], e[r + 1]}, half2v);
                            got = __builtin_amdgcn_fdot2(w[m].h[j], half2v{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)},
                                                         got, false);
                            least = __builtin_elementwise_min(least, w[m].h[j]);
                        }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int d = 0; d < D / 32; ++d) {
                            const half8 value = *reinterpret_cast<const half8*>(values + (d * 4 + m * 2) * kValueRun);
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(value, w[m].v, o[d], 0, 0, 0);
                        }
                    // Weights that f16 holds with fewer than its 11 bits (below 2^-14) go in once more, 2^28 times as
                    // large, and so on down f32's range, less what went in: an output dim whose greatest weights meet
                    // zero codes is as exact as any other. Rare but for rows of extreme scores.
                    const float small = fminf(static_cast<float>(least[0]), static_cast<float>(least[1]));
                    if (__any(small < 0x1p-14f)) {
                        float rest[16];
                        bool more = false;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            rest[r] = e[r] - static_cast<float>(w[r / 4 % 2].h[r / 8 * 2 + r % 4 / 2][r % 2]);
                            rest[r] = e[r] < 0x1p-14f ? rest[r] : 0.0f;
                            more |= rest[r] != 0.0f;
                        }
                        float up = 1.0f;
                        while (__any(more)) {
                            up *= 0x1p28f;
                            more = false;
#pragma unroll
                            for (int m = 0; m < 2; ++m)
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const int r = j / 4 * 8 + m * 4 + j % 4;
                                    const _Float16 x16 = static_cast<_Float16>(rest[r] * up);
                                    w[m].v[j] = x16;
                                    const float left = rest[r] - static_cast<float>(x16) * (1.0f / up);
                                    rest[r] = fabsf(rest[r] * up) < 0x1p-14f ? left : 0.0f;
                                    more |= rest[r] != 0.0f && up < 0x1p100f;
                                }
#pragma unroll
                            for (int d = 0; d < D / 32; ++d) {
                                float16v part = {};
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    const half8 value = *reinterpret_cast<const half8*>(values + (d * 4 + m * 2) * kValueRun);
                                    part = __builtin_amdgcn_mfma_f32_32x32x16_f16(value, w[m].v, part, 0, 0, 0);
                                }
                                o[d] += part * (1.0f / up);
                            }
                        }
                    }
                }
                sum += got == 0.0f ? 0.0f : got / m0.sv[i];
            }
        }
        m0 = m1;
        m1 = m2;
        m2 = m3;
        __syncthreads();
    }

    if (!active) return;
    sum += other_half(sum);
    const int r = w0 + n;
    if (r >= rows) return;
    // o[d][i]: dim 32 d + 8 (i / 4) + 4 half + i % 4 of row r
    if (mine.splits > 1) {
        if (half == 0) {
            p.part_state[(slot * kTile + r - r0) * 2] = ref;
            p.part_state[(slot * kTile + r - r0) * 2 + 1] = sum;
        }
        float* to = p.part_out + (slot * kTile + r - r0) * D + half * 4;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4v*>(to + d * 32 + i * 8) = float4v{o[d][i * 4], o[d][i * 4 + 1], o[d][i * 4 + 2], o[d][i * 4 + 3]};
        return;
    }
    const float over = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(a.out) + (s.row0 + row / p.group) * a.out_row + head * a.out_head + half * 4;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            struct alignas(4 * sizeof(T)) Four {
                T e[4];
            } v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v.e[j] = K::from_f32(sum == 0.0f ? 0.0f : o[d][i * 4 + j] * over);
            if (p.vec_out) {
                *reinterpret_cast<Four*>(out + d * 32 + i * 8) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) out[d * 32 + i * 8 + j] = v.e[j];
            }
        }
}

template <int TYPE, int D>
int launch(const KvAttend& p, hipStream_t stream) {
    const int64_t grid = static_cast<int64_t>(p.row_tiles) * p.slots * p.c.kv_heads;
    if (grid > 0x7fffffff) return kStatusInvalid;
    kv_prompt_kernel<TYPE, D><<<static_cast<unsigned>(grid), 64 * prompt_waves<D>(), 0, stream>>>(p, p.row_tiles);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <int TYPE>
int launch_dim(const KvAttend& p, hipStream_t stream) {
    switch (p.c.head_dim) {
        case 64: return launch<TYPE, 64>(p, stream);
        case 128: return launch<TYPE, 128>(p, stream);
        case 192: return launch<TYPE, 192>(p, stream);
        default: return launch<TYPE, 256>(p, stream);
    }
}

}  // namespace

int kv_prompt_tile(int head_dim) { return head_dim <= 128 ? 256 : 128; }

int launch_kv_prompt(const KvAttend& p, hipStream_t stream) {
    switch (p.a.type) {
        case ROCKNPU_KV_F32: return launch_dim<ROCKNPU_KV_F32>(p, stream);
        case ROCKNPU_KV_F16: return launch_dim<ROCKNPU_KV_F16>(p, stream);
        default: return launch_dim<ROCKNPU_KV_BF16>(p, stream);
    }
}

}  // namespace rk
