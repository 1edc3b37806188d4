// Attention of many rows over the cache: prompts, and pieces of them.
//
// A workgroup of four waves takes a tile of rows of one sequence and kv head
// (the step's tokens times the kv head's heads, so that keys and values serve
// all of them), 32 rows a wave. Blocks pass through LDS one by one: a block's
// codes are converted once per workgroup, into the order in which
// v_mfma_f32_32x32x16 takes them. Scores: keys (32 tokens x 16 dims) times
// queries; a lane ends up with 16 tokens of one row, so maximum and sum are per
// lane but for one exchange, and the weights are the second operand of the next
// product, values (32 dims x 16 tokens) times weights, as they stand.
//
// Per block a wave has 3 D/16 products of 32 cycles (D/16 for the scores, twice
// that for the values, with two parts of a weight; f32 calls 5 D/16); for each of
// a lane's 16 scores a fused multiply-add, an exponential (9 cycles), half a
// maximum, conversion and sum; and its share of the conversion. The matrix and
// vector units overlap because a wave takes block j's maximum and exponentials
// between the products of block j + 1's scores and the conversion of block j + 2
// between the products of block j's values, and because the CU's two workgroups
// are not in step: the wave that is in its products has priority over one that
// works on a maximum or waits for blocks (not with slopes or capped scores, where
// the vector unit is the longer one: 148 against 143 us). Over 4096 rows of 32/8
// heads of 128, bf16, they are busy 42% and 56% of the time; over ragged f32
// prompts with slopes, heads of 64, 19% and 38%, the rest waits and uneven tiles.
// Weights enter as two bf16 (f32 calls: three), which keeps f32's range: as one
// f16 they cost less (165 us where two bf16 take 203), but a row whose greatest
// weights meet zero codes lost the bits of its result below 2^-23 of them. 4096
// rows of 32/8 heads of 128, bf16: 206 us (667 TF/s); 8192 rows: 783 (702 TF/s);
// 4096 rows, f32: 319 us, where the compiler keeps 9 registers in memory.
// Priorities and the maximum between the products took 12 of 180 us off.
#include "kv_attend.h"

namespace rk {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

// The row's reference M follows the maximum only when that grows by more than
// kSlack: rescaling the output costs as much as a block's exponentials, and
// weights, sums and outputs have room for 2^kSlack.
constexpr float kSlack = 30.0f;
// the reference of a row that has seen nothing yet: 2^-inf over it is 0, and so is 2^it over any other
constexpr float kNothing = -1e30f;
// bytes of a 512-byte run of operands in LDS, padded so that the writers' 8
// lanes a cycle meet 8 different 16-byte columns
constexpr int kKeyRun = 528, kValueRun = 544;

constexpr int kWaves = 4, kThreads = 64 * kWaves, kTile = 32 * kWaves;

// This thread's 16-byte pieces of a block.
template <int D>
struct BlockPieces {
    static constexpr int kAll = 2 * kKvBlock * D / 16, kEach = kAll / kThreads;
    uint4 raw[kEach];
};

template <int D>
constexpr int key_bytes() { return D / 8 * kKeyRun; }
template <int D>
constexpr int block_bytes_lds() { return key_bytes<D>() + D / 8 * kValueRun; }

template <int D>
__device__ __forceinline__ void fetch(const uint8_t* pages, int page, BlockPieces<D>& r) {
    const uint8_t* from = pages + static_cast<int64_t>(page) * (64 * D);
#pragma unroll
    for (int i = 0; i < BlockPieces<D>::kEach; ++i)
        r.raw[i] = *reinterpret_cast<const uint4*>(from + (threadIdx.x + i * kThreads) * 16);
}

// The pieces are not used before this.
template <int D>
__device__ __forceinline__ void hold(BlockPieces<D>& r) {
#pragma unroll
    for (int i = 0; i < BlockPieces<D>::kEach; ++i)
        asm volatile("" : "+v"(r.raw[i].x), "+v"(r.raw[i].y), "+v"(r.raw[i].z), "+v"(r.raw[i].w));
}

// Converts piece i into LDS, exactly: keys into f16, values into bf16.
template <int D>
__device__ __forceinline__ void place(const BlockPieces<D>& r, int i, int wave, uint8_t* to) {
    const int piece = threadIdx.x + i * kThreads;
    const uint4 w = r.raw[i];
    constexpr int kKeys = BlockPieces<D>::kAll / 2;
    // whole waves take keys or values, and where a round of the workgroup does, that is known here
    if ((i + 1) * kThreads <= kKeys || (i * kThreads < kKeys && wave * 64 + i * kThreads < kKeys)) {  // keys: token, 16 dims
        uint8_t* p = to + (piece / 128 * 4 + piece % 4) * 2 * kKeyRun + piece / 4 % 32 * 16;
        *reinterpret_cast<half8*>(p) = codes_to_half(w.x, w.y);
        *reinterpret_cast<half8*>(p + kKeyRun) = codes_to_half(w.z, w.w);
    } else {  // values: dims d and d + 16, 8 tokens
        const int v = piece - kKeys;
        uint8_t* p = to + key_bytes<D>() + (v / 64 * 4 + v % 4) * kValueRun + v / 4 % 16 * 16;
        *reinterpret_cast<bhalf8*>(p) = codes_to_bhalf(w.x, w.y);
        *reinterpret_cast<bhalf8*>(p + 256) = codes_to_bhalf(w.z, w.w);
    }
}

// A barrier for what passes through LDS: loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The larger of a row's two lanes' values.
__device__ __forceinline__ float max_of_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) { return x + __shfl_xor(x, 32, 64); }

// PLAIN: neither slopes nor capped scores, whose code costs calls without them 3%
// (170 and 165 us, with weights as f16).
template <int TYPE, int D, bool PLAIN>
__global__ __launch_bounds__(kThreads, (D <= 128 ? 2 : 1)) void kv_prompt_kernel(KvAttend p, int tiles) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    constexpr bool PAIR = TYPE == ROCKNPU_KV_F32;
    constexpr int kParts = PAIR ? 2 : 1, kWeightParts = PAIR ? 3 : 2;
    constexpr int kEarly = 2;             // products of the next block's scores that the maximum is taken between
    constexpr int kAhead = 2;  // operands are read from LDS this many steps before they are used
    constexpr int kSteps = D / 16;  // products of 16 dims of keys, and of values by 32 dims and 16 tokens
    static_assert(kAhead <= kSteps && kEarly < kSteps);
    const rocknpu_kv_cache& c = p.c;
    const rocknpu_kv_attention_args& a = p.a;
    __shared__ alignas(16) uint8_t lds[3][block_bytes_lds<D>()];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The tiles with the most blocks first, a tile's kv heads side by side (one each per XCD where they are 8). Where
    // blocks are shared out tiles have much the same, and the slots that no sequence needs have to be the last workgroups:
    // the GPU deals them out to its engines in turn (512 rows over 8000 tokens, 4 kv heads of 64, f32: 158 us with such
    // slots in between, 107 so; 7 pieces of 33 rows over 5000: 76 and 49; others within 5%).
    const int h = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
    const int slot_at = p.share ? rest / tiles : rest % p.slots;
    const int tile = tiles - 1 - (p.share ? rest % tiles : rest / p.slots);
    const KvSlot mine = kv_slot(p, slot_at);
    const int b = mine.seq;
    if (b < 0) return;
    int lost;
    const KvSpan s = uniform(kv_span(a.past, a.cu, c.dropped, b, static_cast<int>(a.rows), static_cast<int>(a.max_new), lost));
    const int rows = s.n * p.group, r0 = tile * kTile;
    if (r0 >= rows) return;
    kv_leave_slot(p, mine, h, tile);
    const int total = s.past + s.n, gone = uniform(lost);
    const int held = min((total + kKvBlock - 1) / kKvBlock - gone, c.max_blocks);
    const int prefix = uniform(kv_prefix(a, b));
    const int64_t entry_row = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks;
    const KvRange range = kv_range(a, c.starts + entry_row, held, gone, s.past + r0 / p.group,
                                   s.past + (min(r0 + kTile, rows) - 1) / p.group, prefix);
    const int count = range.count();
    const int chunk = (count + mine.splits - 1) / mine.splits;
    const int begin = mine.split * chunk, end = min(begin + chunk, count);
    const int64_t slot = (static_cast<int64_t>(h) * p.row_tiles + tile) * p.slots + slot_at;
    if (begin >= end && mine.splits > 1) {
        if (tid < kTile) reinterpret_cast<float2*>(p.part_state)[slot * kTile + tid] = make_float2(-__builtin_inff(), 0.0f);
        return;
    }

    // The wave's rows are w0 + n. A row sees [low, low + span] and what lies before `pre`; `full` and `some`: what every
    // row and some row of the wave sees.
    const int w0 = r0 + wave * 32;
    const bool active = w0 < rows, windowed = a.window != 0;
    const int q0 = s.past + min(w0, rows - 1) / p.group, q1 = s.past + (min(w0 + 32, rows) - 1) / p.group;
    const int pre = min(prefix, total), newest = total - 1;
    const int full_low = windowed ? max(q1 - a.window + 1, 0) : 0, full_high = a.causal ? min(q0, newest) : newest;
    const int some_low = windowed ? max(q0 - a.window + 1, 0) : 0, some_high = a.causal ? min(q1, newest) : newest;
    const int row = min(w0 + n, rows - 1), head = h * p.group + row % p.group, qpos = s.past + row / p.group;
    const int low = windowed ? max(qpos - a.window + 1, 0) : 0;
    const unsigned span = static_cast<unsigned>((a.causal ? min(qpos, newest) : newest) - low);
    const float slope = !PLAIN && a.slopes ? a.slopes[head] : 0.0f;
    // Block j of the workgroup's part: its bytes are loaded in iteration j - 4 (a trip to memory takes longer than an
    // iteration) and go to LDS in iteration j - 2. Page numbers, positions and scales are looked up 64 blocks at a time, a
    // block per lane, half a batch ahead. (Looked up block by block they were what an iteration waited for: 4096 tokens,
    // 32/8 heads of 128, bf16: 197 us; 180 with this and rows stored whole.)
    struct Batch {
        int page, start;
        float sk, sv;
    };
    struct Meta {
        int start;
        float sk, sv;
    };
    const int32_t* table = c.table + entry_row;
    const int32_t* starts = c.starts + entry_row;
    const int blocks = end - begin;
    Batch batch{}, batch_1{};  // of blocks base .. base + 63, and of the next 64
    int base = 0;
    const auto look_up = [&](int first, Batch& r) {
        if (first + lane < blocks) {
            const int at = range.entry(begin + first + lane);
            r.page = table[at];
            r.start = starts[at];
        }
    };
    const auto look_up_scales = [&](int first, Batch& r) {
        const bool ok = r.page >= 0 && r.page < c.n_pages;
        r.page = ok ? r.page : 0;
        if (first + lane < blocks) {
            const float2 x = reinterpret_cast<const float2*>(c.scales)[r.page];
            r.sk = kv_scale(x.x, ok);
            r.sv = kv_scale(x.y, ok);
        }
    };
    // a field of block j, for base <= j < base + 128; past the end what it is does not matter, but it is a page that exists
    const auto of_block = [&](int j, int here, int there) {
        return j - base < 64 ? __builtin_amdgcn_readlane(here, j - base) : __builtin_amdgcn_readlane(there, j - base - 64);
    };
    const auto meta_of = [&](int j) {
        return Meta{of_block(j, batch.start, batch_1.start),
                    __uint_as_float(of_block(j, __float_as_uint(batch.sk), __float_as_uint(batch_1.sk))),
                    __uint_as_float(of_block(j, __float_as_uint(batch.sv), __float_as_uint(batch_1.sv)))};
    };
    const auto fetch_block = [&](int j, BlockPieces<D>& r) { fetch<D>(c.pages, of_block(j, batch.page, batch_1.page), r); };

    BlockPieces<D> even, odd;
    look_up(0, batch);
    half8 q[kParts][kSteps];
    float unit;  // a product's weight in the score
    {
        const T* src = static_cast<const T*>(a.q) + (s.row0 + row / p.group) * a.q_row + head * a.q_head + half * 8;
        float x[kSteps][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) load8<TYPE>(src + i * 16, p.vec_q, x[i]);
        // the first blocks' bytes, whose pages are known by now, come while the queries are worked on
        look_up_scales(0, batch);
        fetch_block(0, even);
        fetch_block(1, odd);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
        const float power = row_power(max_of_halves(top));
        // the queries take the scale's sign, so that scores rise with their products
        unit = fabsf(a.scale) / power;
        const float signed_power = a.scale < 0.0f ? -power : power;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[i][e] * signed_power;
                q[0][i][e] = static_cast<_Float16>(v);
                if constexpr (PAIR) q[1][i][e] = static_cast<_Float16>(v - static_cast<float>(q[0][i][e]));
            }
    }

    float16v o[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) o[d] = float16v{};
    float ref = kNothing, sum = 0.0f;

    // operand k of the scores' products (16 dims), and of the values': all tiles of 32 dims with 16 of the tokens, then with
    // the others
    const auto read_key = [&](const uint8_t* at, int k) {
        return *reinterpret_cast<const half8*>(at + half * kKeyRun + n * 16 + k * 2 * kKeyRun);
    };
    const auto read_value = [&](const uint8_t* at, int k) {
        return *reinterpret_cast<const bhalf8*>(at + key_bytes<D>() + half * kValueRun + n * 16 +
                                               (k % (kSteps / 2) * 2 + k / (kSteps / 2)) * 2 * kValueRun);
    };
    // x[r]: token 8 (r / 4) + 4 half + r % 4 of the block, row n
    const auto product = [&](const half8& key, int k, float16v& x) {
#pragma unroll
        for (int part = 0; part < kParts; ++part) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, q[part][k], x, 0, 0, 0);
    };

    Meta meta{}, meta_1{};  // of blocks j, j + 1
    int now = 0;            // block j is in lds[now], block j + 1 in the next buffer
    // Iteration j: x holds block j's products, x_1 takes block j + 1's; `two` holds block j + 2 and takes block j + 4.
    const auto iterate = [&](int j, float16v& x, float16v& x_1, BlockPieces<D>& two) {
        const int then = now == 2 ? 0 : now + 1, later = then == 2 ? 0 : then + 1;
        const uint8_t* at = lds[now];
        const uint8_t* at_1 = lds[then];
        const float sk = meta.sk, sv = meta.sv;
        const bool before = meta.start + kKvBlock <= pre;
        const bool any = active && ((meta.start <= some_high && meta.start + kKvBlock > some_low) || meta.start < pre);
        x_1 = float16v{};
        half8 key[kSteps];
        bhalf8 value[kSteps];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) key[k] = read_key(at_1, k);
        // operand k + kAhead of the scores' products, behind them the first of the values'
        const auto read_ahead = [&](int k) {
            if (k + kAhead < kSteps)
                key[k + kAhead] = read_key(at_1, k + kAhead);
            else
                value[k + kAhead - kSteps] = read_value(at, k + kAhead - kSteps);
        };
        if (__builtin_expect(any, 1)) {
            // scores to exponents over the row's reference, which follows the maximum
            const bool folds = kv_folds(sv);
            const float lift = __log2f(folds ? sv : kKvFoldLeast);
            float inverse = __builtin_amdgcn_rcpf(sv);
            float factor = unit * sk * kLog2e, off = lift, most;
            const bool full = before || (meta.start >= full_low && meta.start + kKvBlock - 1 <= full_high);
            if (__builtin_expect(full && PLAIN, 1)) {
                float m[kEarly];
#pragma unroll
                for (int k = 0; k < kEarly; ++k) {
                    read_ahead(k);
                    product(key[k], k, x_1);
                    m[k] = x[k * (16 / kEarly)];
#pragma unroll
                    for (int r = 1; r < 16 / kEarly; ++r) m[k] = fmaxf(m[k], x[k * (16 / kEarly) + r]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                most = m[0];
#pragma unroll
                for (int k = 1; k < kEarly; ++k) most = fmaxf(most, m[k]);
                most = __builtin_fmaf(most, factor, off);
                __builtin_amdgcn_s_setprio(1);
            } else if (!PLAIN && full && a.softcap == 0.0f) {
                // a distance's share of the exponent is the block's plus a multiple of the slope (5 prompts of up to 1500
                // tokens, 32/4 heads of 64, f32: 102 us, with the general form's operations 143)
                const float rise = slope * kLog2e;
                const float at_0 = __builtin_fmaf(rise, static_cast<float>(meta.start + half * 4 - qpos), off);
                most = kNothing;
#pragma unroll
                for (int k = 0; k < kEarly; ++k) {
                    read_ahead(k);
                    product(key[k], k, x_1);
#pragma unroll
                    for (int r = k * (16 / kEarly); r < (k + 1) * (16 / kEarly); ++r) {
                        x[r] = __builtin_fmaf(x[r], factor, __builtin_fmaf(rise, static_cast<float>(r / 4 * 8 + r % 4), at_0));
                        most = fmaxf(most, x[r]);
                    }
                }
                factor = 1.0f;
                off = 0.0f;
            } else {
#pragma unroll
                for (int k = 0; k < kEarly; ++k) {
                    read_ahead(k);
                    product(key[k], k, x_1);
                }
                most = kNothing;
                const float to_score = PLAIN ? factor : unit * sk;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int kpos = meta.start + r / 4 * 8 + half * 4 + r % 4;
                    float y = x[r] * to_score;
                    if constexpr (!PLAIN) {
                        if (a.softcap != 0.0f) y = kv_cap<PAIR>(y, a.softcap);
                        if (a.slopes) y += slope * static_cast<float>(kpos - qpos);
                        y *= kLog2e;
                    }
                    x[r] = static_cast<unsigned>(kpos - low) <= span || kpos < pre ? y + lift : -__builtin_inff();
                    most = fmaxf(most, x[r]);
                }
                factor = 1.0f;
                off = 0.0f;
            }
            most = max_of_halves(most);
            if (__builtin_expect(__any(most > ref + kSlack || !folds), 0)) {
                const float to = fmaxf(ref, most);
                const float keep = exp2_fast(ref - to);
                ref = to;
                sum *= keep;
#pragma unroll
                for (int d = 0; d < D / 32; ++d) o[d] *= keep;
                if (!folds) {
                    float apart = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) apart += exp2_fast(__builtin_fmaf(x[r], factor, off - ref));
                    sum += apart / kKvFoldLeast;
                    inverse = 0.0f;
                    off += __log2f(sv / kKvFoldLeast);
                }
            }
            off -= ref;

            // the next block's scores, and between them this one's weights
#pragma unroll
            for (int k = kEarly; k < kSteps; ++k) {
                read_ahead(k);
                product(key[k], k, x_1);
#pragma unroll
                for (int e = 16 * (k - kEarly) / (kSteps - kEarly); e < 16 * (k + 1 - kEarly) / (kSteps - kEarly); ++e)
                    x[e] = exp2_fast(__builtin_fmaf(x[e], factor, off));
            }
            bhalf8 w[2][kWeightParts];
            float got = 0.0f;
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                float part[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    part[i] = x[i / 4 * 8 + h2 * 4 + i % 4];
                    got += part[i];
                }
                split_bhalf(part, w[h2]);
            }
            sum += got == 0.0f ? 0.0f : got * inverse;
            // Values times weights, and between them the later block's conversion. Its bytes are first touched here: moved
            // up, the conversion would wait for them at the iteration's start.
            if constexpr (PLAIN) __builtin_amdgcn_s_setprio(2);
            __builtin_amdgcn_sched_barrier(0);
            hold<D>(two);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const int h2 = k / (kSteps / 2), d = k % (kSteps / 2);
                if (k + kAhead < kSteps) value[k + kAhead] = read_value(at, k + kAhead);
#pragma unroll
                for (int part = 0; part < kWeightParts; ++part)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value[k], w[h2][part], o[d], 0, 0, 0);
                if (k % (kSteps / BlockPieces<D>::kEach) == 0)
                    place<D>(two, k / (kSteps / BlockPieces<D>::kEach), wave, lds[later]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) product(k < kAhead ? key[k] : read_key(at_1, k), k, x_1);
            hold<D>(two);
#pragma unroll
            for (int i = 0; i < BlockPieces<D>::kEach; ++i) place<D>(two, i, wave, lds[later]);
        }
        if constexpr (PLAIN) __builtin_amdgcn_s_setprio(0);
        meta = meta_1;
        meta_1 = meta_of(j + 2);
        fetch_block(j + 4, two);
        if (j + 1 - base == 32) look_up(base + 64, batch_1);
        if (j + 1 - base == 48) look_up_scales(base + 64, batch_1);
        if (j + 1 - base == 64) {
            batch = batch_1;
            base += 64;
        }
        now = then;
        lds_barrier();
    };

    float16v x = {}, x_1;
    if (blocks > 0) {
        // blocks 0 and 1 into LDS, blocks 2 and 3 on their way
        meta = meta_of(0);
        meta_1 = meta_of(1);
#pragma unroll
        for (int i = 0; i < BlockPieces<D>::kEach; ++i) place<D>(even, i, wave, lds[0]);
        fetch_block(2, even);
#pragma unroll
        for (int i = 0; i < BlockPieces<D>::kEach; ++i) place<D>(odd, i, wave, lds[1]);
        fetch_block(3, odd);
    }
    lds_barrier();
    if (blocks > 0) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) product(read_key(lds[0], k), k, x);
    }
    for (int j = 0; j < blocks; j += 2) {
        iterate(j, x, x_1, even);
        if (j + 1 < blocks) iterate(j + 1, x_1, x, odd);
    }

    if (!active) return;
    sum = sum_of_halves(sum);
    const int r = w0 + n;
    // o[d][i]: dim 32 d + 8 (i / 4) + 4 half + i % 4 of row r
    if (mine.splits > 1) {
        if (r >= rows) return;
        if (half == 0) reinterpret_cast<float2*>(p.part_state)[slot * kTile + r - r0] = make_float2(ref, sum);
        float* to = p.part_out + (slot * kTile + r - r0) * D + half * 4;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4v*>(to + d * 32 + i * 8) =
                    float4v{o[d][i * 4], o[d][i * 4 + 1], o[d][i * 4 + 2], o[d][i * 4 + 3]};
        return;
    }
    const float over = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(a.out);
    if (!PAIR && p.vec_out) {
        // through LDS, so that whole rows are stored, 16 bytes a lane
        constexpr int kRow = D + 8;  // elements, padded
        T* rows_lds = reinterpret_cast<T*>(&lds[0][0]) + wave * 32 * kRow;
        static_assert(PAIR || kWaves * 32 * kRow * 2 <= 3 * block_bytes_lds<D>());
        struct alignas(8) Four {
            T e[4];
        };
        struct alignas(16) Eight {
            T e[16 / sizeof(T)];
        };
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                Four v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v.e[e] = K::from_f32(sum == 0.0f ? 0.0f : o[d][i * 4 + e] * over);
                *reinterpret_cast<Four*>(rows_lds + n * kRow + d * 32 + i * 8 + half * 4) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
#pragma unroll
        for (int i = 0; i < 32 * D / 8 / 64; ++i) {
            const int at = i * 64 + lane, m = at / (D / 8), d = at % (D / 8) * 8, rr = w0 + m;
            if (rr < rows)
                *reinterpret_cast<Eight*>(out + (s.row0 + rr / p.group) * a.out_row + (h * p.group + rr % p.group) * a.out_head + d) =
                    *reinterpret_cast<Eight*>(rows_lds + m * kRow + d);
        }
        return;
    }
    if (r >= rows) return;
    out += (s.row0 + row / p.group) * a.out_row + head * a.out_head + half * 4;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            struct alignas(4 * sizeof(T)) Four {
                T e[4];
            } v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v.e[e] = K::from_f32(sum == 0.0f ? 0.0f : o[d][i * 4 + e] * over);
            if (p.vec_out) {
                *reinterpret_cast<Four*>(out + d * 32 + i * 8) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) out[d * 32 + i * 8 + e] = v.e[e];
            }
        }
}

template <int TYPE, int D>
int launch(const KvAttend& p, hipStream_t stream) {
    const int64_t grid = static_cast<int64_t>(p.row_tiles) * p.slots * p.c.kv_heads;
    if (grid > 0x7fffffff) return kStatusInvalid;
    if (p.a.softcap == 0.0f && !p.a.slopes)
        kv_prompt_kernel<TYPE, D, true><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p, p.row_tiles);
    else
        kv_prompt_kernel<TYPE, D, false><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p, p.row_tiles);
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

int kv_prompt_tile() { return kTile; }

int launch_kv_prompt(const KvAttend& p, hipStream_t stream) {
    switch (p.a.type) {
        case ROCKNPU_KV_F32: return launch_dim<ROCKNPU_KV_F32>(p, stream);
        case ROCKNPU_KV_F16: return launch_dim<ROCKNPU_KV_F16>(p, stream);
        default: return launch_dim<ROCKNPU_KV_BF16>(p, stream);
    }
}

}  // namespace rk
