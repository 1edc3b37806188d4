// Attention of few rows over a long cache: the cache streams through the matrix
// units once for up to 16 rows (a kv head's heads times the step's tokens).
//
// A workgroup of four or eight waves takes one split of a (sequence, kv head, tile
// of 16 rows), its waves the split's blocks in turn. Blocks come from memory straight into
// the operand registers (whole 1 KiB runs per load, the next block's loads in
// flight behind the current one's work), so LDS is used only to join the waves.
// Scores: keys (16 tokens x 32 dims) times the rows' queries; they leave in the
// layout in which the next product takes weights: values (16 dims x 32 tokens)
// times weights. Bound by the cache's bytes: one row of two sequences of 100000
// tokens, 8 kv heads of 128, 420 MB in 79 us (5.3 TB/s, above a large copy's 4.7);
// by the longest part where lengths differ: 32 of 500-4100 tokens, 145 MB in 38.
#include "kv_attend.h"

namespace rk {
namespace {

template <int D>
struct BlockRegs {
    uint4 k[2][D / 64];  // token tile, 64 dims
    uint4 v[D / 32];
};

template <int D>
__device__ __forceinline__ void load_block(const uint8_t* pages, int64_t page, int lane, BlockRegs<D>& r) {
    const uint8_t* keys = pages + page * (2 * kKvBlock * D) + lane % 16 * 64 + lane / 16 * 16;
    const uint8_t* values = pages + page * (2 * kKvBlock * D) + kKvBlock * D + lane % 16 * 64 + lane / 16 * 16;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) r.k[t][c] = *reinterpret_cast<const uint4*>(keys + (c * 32 + t * 16) * 64);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) r.v[c] = *reinterpret_cast<const uint4*>(values + c * 1024);
}

__device__ __forceinline__ float max_over_quads(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_over_quads(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// Queries enter as f16, those of f32 calls as hi + lo; weights as two bf16, those
// of f32 calls as three, which keeps f32's range: an output dim whose greatest
// weights meet zero codes is as exact as any other.
template <int TYPE, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void kv_stream_kernel(KvAttend p) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    constexpr bool PAIR = TYPE == ROCKNPU_KV_F32;
    constexpr int kParts = PAIR ? 2 : 1, kWeightParts = PAIR ? 3 : 2;
    const rocknpu_kv_cache& c = p.c;
    const rocknpu_kv_attention_args& a = p.a;
    __shared__ float state[WAVES][kKvTileRows][2];
    __shared__ alignas(16) float sums[WAVES][kKvTileRows][D + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane % 16, quad = lane / 16;
    // Slots that no sequence needs are the last workgroups: the GPU deals workgroups out to its engines in turn, and with
    // such slots in between one engine gets more work than it holds while others wait (64 rows a kv head over 16000
    // tokens 38 us instead of 22).
    const int h = blockIdx.x, tile = blockIdx.y, slot_at = blockIdx.z;
    const KvSlot mine = kv_slot(p, slot_at);
    const int b = mine.seq;
    if (b < 0) return;
    const int kept = kv_prefix(a, b);
    int lost;
    const KvSpan s = uniform(kv_span(a.past, a.cu, c.dropped, b, static_cast<int>(a.rows), static_cast<int>(a.max_new), lost));
    const int rows = s.n * p.group, r0 = tile * kKvTileRows;
    const int total = s.past + s.n, gone = uniform(lost), prefix = uniform(kept);
    if (r0 >= rows) return;
    kv_leave_slot(p, mine, h, tile);
    const int held = min((total + kKvBlock - 1) / kKvBlock - gone, c.max_blocks);
    const int64_t entry_row = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks;
    const int q0 = s.past + r0 / p.group, q1 = s.past + (min(r0 + kKvTileRows, rows) - 1) / p.group;
    const KvRange range = kv_range(a, c.starts + entry_row, held, gone, q0, q1, prefix);
    const int count = range.count();
    const int chunk = (count + mine.splits - 1) / mine.splits;
    const int begin = mine.split * chunk, end = min(begin + chunk, count);
    const int64_t slot = (static_cast<int64_t>(h) * p.row_tiles + tile) * p.slots + slot_at;
    if (begin >= end && mine.splits > 1) {
        if (tid < kKvTileRows) {
            p.part_state[(slot * kKvTileRows + tid) * 2] = -__builtin_inff();
            p.part_state[(slot * kKvTileRows + tid) * 2 + 1] = 0.0f;
        }
        return;
    }

    // Lane l looks up the wave's l-th block from `base` on. The first blocks are looked up and their bytes asked for before
    // the queries are converted: the chain of trips to memory is what a short context waits for.
    int my_page = 0, my_start = 0;
    float my_sk = 0.0f, my_sv = 0.0f;
    BlockRegs<D> next;
    const auto look_up = [&](int base) {
        const int nth = base + lane * WAVES + wave;
        if (nth < end) {
            const int at = range.entry(nth);
            my_page = c.table[entry_row + at];
            my_start = c.starts[entry_row + at];
        }
    };
    const auto blocks_from = [&](int base) { return (min(end - base, 64 * WAVES) - wave + WAVES - 1) / WAVES; };
    const auto fetch_first = [&](int base) {
        const bool ok = my_page >= 0 && my_page < c.n_pages;
        my_page = ok ? my_page : 0;
        if (base + lane * WAVES + wave < end) {
            const float2 sc = reinterpret_cast<const float2*>(c.scales)[my_page];
            my_sk = kv_scale(sc.x, ok);
            my_sv = kv_scale(sc.y, ok);
        }
        if (blocks_from(base) > 0) load_block<D>(c.pages, __builtin_amdgcn_readlane(my_page, 0), lane, next);
    };
    if (begin < end) look_up(begin);

    // this lane's row: column n of the products
    const int row = min(r0 + n, rows - 1), head = h * p.group + row % p.group;
    const int qpos = s.past + row / p.group;
    half8 q[kParts][D / 32];
    float unit;  // score per unit of (query as held) . (key codes), without the key scale
    {
        const T* src = static_cast<const T*>(a.q) + (s.row0 + row / p.group) * a.q_row + head * a.q_head;
        float x[D / 32][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) load8<TYPE>(src + i / 2 * 64 + quad * 16 + i % 2 * 8, p.vec_q, x[i]);
        if (begin < end) fetch_first(begin);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
        const float power = row_power(max_over_quads(top));
        unit = a.scale / power;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[i][e] * power;
                q[0][i][e] = static_cast<_Float16>(v);
                if constexpr (PAIR) q[1][i][e] = static_cast<_Float16>(v - static_cast<float>(q[0][i][e]));
            }
    }
    const float slope = a.slopes ? a.slopes[head] : 0.0f;

    float top = -__builtin_inff(), sum = 0.0f;
    float4v o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = float4v{0, 0, 0, 0};

    for (int base = begin; base < end; base += 64 * WAVES) {
        if (base != begin) {
            look_up(base);
            fetch_first(base);
        }
        const int here = blocks_from(base);  // the wave's blocks
        for (int k = 0; k < here; ++k) {
            const BlockRegs<D> cur = next;
            if (k + 1 < here) load_block<D>(c.pages, __builtin_amdgcn_readlane(my_page, k + 1), lane, next);
            const int start = __builtin_amdgcn_readlane(my_start, k);
            const float sk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_sk), k));
            const float sv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_sv), k));
            float4v x[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                x[t] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint4 raw = cur.k[t][i / 2];
                    const half8 key = i % 2 ? codes_to_half(raw.z, raw.w) : codes_to_half(raw.x, raw.y);
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, q[part][i], x[t], 0, 0, 0);
                }
            }
            // scores in powers of two: x[t][i] is token 16 t + 4 quad + i
            const bool plain = a.softcap == 0.0f && !a.slopes;
            float factor = unit * sk * kLog2e;
            if (!plain) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float y = x[t][i] * (unit * sk);
                        if (a.softcap != 0.0f) y = kv_cap<PAIR>(y, a.softcap);
                        if (a.slopes) y += slope * static_cast<float>(start + t * 16 + quad * 4 + i - qpos);
                        x[t][i] = y;
                    }
                factor = kLog2e;
            }
            const bool folds = kv_folds(sv);
            const float lift = __log2f(folds ? sv : kKvFoldLeast);
            float most = -__builtin_inff();
            const bool folded = !kv_all_seen(a, start, q0, q1, prefix, total);
            if (!folded) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = fmaxf(most, __builtin_fmaf(x[t][i], factor, lift));
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = kv_seen(a, start + t * 16 + quad * 4 + i, qpos, prefix, total);
                        // a masked score is -inf whatever its factor: NaN and the sign of `factor` included
                        x[t][i] = seen ? __builtin_fmaf(x[t][i], factor, lift) : -__builtin_inff();
                        most = fmaxf(most, x[t][i]);
                    }
                factor = 1.0f;
            }
            most = max_over_quads(most);
            const float now = fmaxf(top, most);
            const float ref = now == -__builtin_inff() ? 0.0f : now;
            float shift = (folded ? 0.0f : lift) - ref, apart = 0.0f;
            if (__any(now != top || !folds)) {
                const float keep = exp2_fast(top - ref);
                sum *= keep;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[i] *= keep;
                top = now;
                if (!folds) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) apart += exp2_fast(__builtin_fmaf(x[t][i], factor, shift));
                    apart /= kKvFoldLeast;
                    shift += __log2f(sv / kKvFoldLeast);
                }
            }
            float e[8], got = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[t * 4 + i] = exp2_fast(__builtin_fmaf(x[t][i], factor, shift));
                    got += e[t * 4 + i];
                }
            bhalf8 w[kWeightParts];
            split_bhalf(e, w);
            got = !folds ? apart : got == 0.0f ? 0.0f : got / sv;
            sum += got;
            if (p.block_sums) {
                const float all = sum_over_quads(got);
                if (quad == 0 && r0 + n < rows) {
                    const int64_t at = (entry_row + range.entry(base + k * WAVES + wave)) * (p.row_tiles * kKvTileRows) + r0 + n;
                    reinterpret_cast<float2*>(p.block_sums)[at] = make_float2(all, ref);
                }
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint4 raw = cur.v[i / 2];
                const bhalf8 value = i % 2 ? codes_to_bhalf(raw.z, raw.w) : codes_to_bhalf(raw.x, raw.y);
#pragma unroll
                for (int part = 0; part < kWeightParts; ++part)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, w[part], o[i], 0, 0, 0);
            }
        }
    }

    // join the waves
    sum = sum_over_quads(sum);
    if (quad == 0) {
        state[wave][n][0] = top;
        state[wave][n][1] = sum;
    }
    __syncthreads();
    float most = state[0][n][0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) most = fmaxf(most, state[w][n][0]);
    const float ref = most == -__builtin_inff() ? 0.0f : most;
    const float keep = exp2_fast(top - ref);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<float4v*>(&sums[wave][n][i * 16 + quad * 4]) = o[i] * keep;
    __syncthreads();
    for (int i = tid; i < kKvTileRows * D / 4; i += 64 * WAVES) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (r0 + r >= rows) break;
        float4v acc = *reinterpret_cast<float4v*>(&sums[0][r][d]);
        float m = state[0][r][0], l = 0.0f;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            acc += *reinterpret_cast<float4v*>(&sums[w][r][d]);
            m = fmaxf(m, state[w][r][0]);
        }
        const float at = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) l += state[w][r][1] * exp2_fast(state[w][r][0] - at);
        if (mine.splits > 1 || p.block_sums) {
            if (d == 0) {
                p.part_state[(slot * kKvTileRows + r) * 2] = m;
                p.part_state[(slot * kKvTileRows + r) * 2 + 1] = l;
            }
        }
        if (mine.splits > 1) {
            *reinterpret_cast<float4v*>(p.part_out + (slot * kKvTileRows + r) * D + d) = acc;
        } else {
            const int rr = r0 + r, hd = h * p.group + rr % p.group;
            T* out = static_cast<T*>(a.out) + (s.row0 + rr / p.group) * a.out_row + hd * a.out_head + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = K::from_f32(l == 0.0f ? 0.0f : acc[e] / l);
        }
    }
}

// Joins the splits of a tile's rows: the first workgroups take 4 / WAVES rows
// each, a row's splits read side by side, the others (with block weights) a block
// per thread. A row of many splits takes a workgroup, so that its loads are all
// in flight together; of few, a wave (2048 rows of 8 heads in 2 splits: a
// workgroup each took 45 us).
template <int TYPE, int D, int WAVES>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttend p, int row_groups) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    constexpr int kPer = D / 4;         // lanes that read a split's row
    constexpr int kBeside = 64 / kPer;  // splits that a wave reads side by side
    const rocknpu_kv_cache& c = p.c;
    const rocknpu_kv_attention_args& a = p.a;
    __shared__ float final_state[kKvMaxWeightRows][2];
    __shared__ float keep[4 / WAVES][kKvMaxSplits];
    __shared__ alignas(16) float part[WAVES][D];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = blockIdx.y, b = blockIdx.z;
    int lost;
    const KvSpan s = uniform(kv_span(a.past, a.cu, c.dropped, b, static_cast<int>(a.rows), static_cast<int>(a.max_new), lost));
    const int rows = s.n * p.group;
    const int64_t seq = static_cast<int64_t>(b) * c.kv_heads + h;
    const bool joins = static_cast<int>(blockIdx.x) < row_groups;
    if (joins && static_cast<int>(blockIdx.x) * (4 / WAVES) >= rows) return;
    // A sequence without rows has no slots, and left none. What was left is held to the workspace's bounds: lengths that
    // change under a call (a caller's missing wait) may leave a sequence here whose slots nothing wrote.
    const int2 slots = p.share && rows > 0 ? p.slots_of[b] : make_int2(b, 1);
    const int first = uniform(min(max(slots.x, 0), p.slots - 1));
    const int splits = uniform(min(max(slots.y, 1), min(p.slots - first, kKvMaxSplits)));
    const auto slot_of = [&](int r) { return (static_cast<int64_t>(h) * p.row_tiles + r / p.tile_rows) * p.slots + first; };
    const auto state_of = [&](int r) {
        return reinterpret_cast<const float2*>(p.part_state) + slot_of(r) * p.tile_rows + r % p.tile_rows;
    };
    if (joins) {
        const int r = blockIdx.x * (4 / WAVES) + wave / WAVES, nth = wave % WAVES, mine = wave / WAVES;
        if (splits <= 1) return;  // its only workgroup wrote the row
        float4v acc = {0, 0, 0, 0};
        if (r < rows) {
            const float2* st = state_of(r);
            float most = -__builtin_inff(), total = 0.0f;
            float2 state[kKvMaxSplits / 64];
#pragma unroll
            for (int k = 0; k < kKvMaxSplits / 64; ++k) {
                const int i = k * 64 + lane;
                state[k] = i < splits ? st[i * p.tile_rows] : make_float2(-__builtin_inff(), 0.0f);
                most = fmaxf(most, state[k].x);
            }
            most = wave_max(most);
            const float ref = most == -__builtin_inff() ? 0.0f : most;
#pragma unroll
            for (int k = 0; k < kKvMaxSplits / 64; ++k) total += state[k].y * exp2_fast(state[k].x - ref);
#pragma unroll
            for (int g = 32; g >= 1; g >>= 1) total += __shfl_xor(total, g, 64);
            // a split without blocks wrote no sums: its factor is 0 and its sums are not read
#pragma unroll
            for (int k = 0; k < kKvMaxSplits / 64; ++k)
                if (k * 64 + lane < splits)
                    keep[mine][k * 64 + lane] = state[k].y == 0.0f ? 0.0f : exp2_fast(state[k].x - ref) / total;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
            const int beside = lane / kPer;
            const float* from = p.part_out + (slot_of(r) * p.tile_rows + r % p.tile_rows) * D + lane % kPer * 4;
            if (beside < kBeside) {
#pragma unroll 4
                for (int i = nth * kBeside + beside; i < splits; i += WAVES * kBeside) {
                    const float f = keep[mine][i];
                    if (f != 0.0f) acc += f * *reinterpret_cast<const float4v*>(from + static_cast<int64_t>(i) * p.tile_rows * D);
                }
            }
#pragma unroll
            for (int g = kPer; g < 64 && kBeside > 1; g *= 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], g, 64);
        }
        if constexpr (WAVES > 1) {
            if (lane < kPer) *reinterpret_cast<float4v*>(&part[nth][lane * 4]) = acc;
            __syncthreads();
            if (nth > 0) return;
#pragma unroll
            for (int w = 1; w < WAVES; ++w)
                if (lane < kPer) acc += *reinterpret_cast<float4v*>(&part[w][lane * 4]);
        }
        if (r < rows && lane < kPer) {
            const int hd = h * p.group + r % p.group;
            T* out = static_cast<T*>(a.out) + (s.row0 + r / p.group) * a.out_row + hd * a.out_head + lane * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = K::from_f32(acc[e]);
        }
        return;
    }
    // The rows' maxima and sums over their splits, all rows at once: as many lanes a row as there are (rows one after the
    // other: 64 rows of 8 splits with 501 blocks 34 us instead of 17).
    int lanes = 64;
    while (lanes > 1 && 256 / lanes < rows) lanes /= 2;
    {
        const int r = tid / lanes, l = tid % lanes;
        const float2* st = state_of(min(r, max(rows - 1, 0)));
        const int n = r < rows ? splits : 0;
        float most = -__builtin_inff(), total = 0.0f;
#pragma unroll 4
        for (int i = l; i < n; i += lanes) most = fmaxf(most, st[i * p.tile_rows].x);
        for (int o = lanes / 2; o >= 1; o /= 2) most = fmaxf(most, __shfl_xor(most, o, 64));
        const float ref = most == -__builtin_inff() ? 0.0f : most;
#pragma unroll 4
        for (int i = l; i < n; i += lanes) total += st[i * p.tile_rows].y * exp2_fast(st[i * p.tile_rows].x - ref);
        for (int o = lanes / 2; o >= 1; o /= 2) total += __shfl_xor(total, o, 64);
        if (l == 0 && r < rows) {
            final_state[r][0] = ref;
            final_state[r][1] = total;
        }
    }
    __syncthreads();
    const int at = (blockIdx.x - row_groups) * 256 + tid;
    if (at >= c.max_blocks) return;
    const int64_t entry = seq * c.max_blocks + at;
    float got = 0.0f;
    const int total = s.past + s.n, gone = uniform(lost);
    if (at < min((total + kKvBlock - 1) / kKvBlock - gone, c.max_blocks)) {
        const int start = c.starts[entry], prefix = uniform(kv_prefix(a, b));
        for (int tile = 0; tile * p.tile_rows < rows; ++tile) {
            const int r0 = tile * p.tile_rows, r1 = min(r0 + p.tile_rows, rows);
            // the blocks that kv_range gave the tile
            const int q0 = s.past + r0 / p.group, q1 = s.past + (r1 - 1) / p.group;
            if (a.causal && start >= prefix &&
                (start > q1 || (a.window != 0 && start + kKvBlock <= q0 - a.window + 1)))
                continue;
            const float2* sums = reinterpret_cast<const float2*>(p.block_sums) + entry * (p.row_tiles * p.tile_rows);
#pragma unroll
            for (int g = 0; g < kKvTileRows; g += 4) {
                if (r0 + g >= r1) break;
                float2 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = sums[r0 + g + i];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r0 + g + i < r1 && x[i].x != 0.0f)
                        got += x[i].x * exp2_fast(x[i].y - final_state[r0 + g + i][0]) / final_state[r0 + g + i][1];
            }
        }
    }
    a.weights_out[entry] = c.weights[entry] + got;
}

template <int TYPE, int D>
int launch(const KvAttend& p, hipStream_t stream) {
    const dim3 grid(p.c.kv_heads, p.row_tiles, p.slots);
    if (p.a.rows > 0 && p.a.max_new > 0) {
        if constexpr (D != 256) {
            if (p.waves == 8) kv_stream_kernel<TYPE, D, 8><<<grid, 512, 0, stream>>>(p);
        }
        if constexpr (D != 192) {
            if (p.waves == 4) kv_stream_kernel<TYPE, D, 4><<<grid, 256, 0, stream>>>(p);
        }
    }
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <int TYPE, int D>
int launch_join(const KvAttend& p, hipStream_t stream) {
    // a sequence's splits are about share / batch
    const bool many = p.share > 12 * p.c.batch;
    const int rows = p.part_out ? static_cast<int>(p.a.max_new) * p.group : 0;
    const int row_groups = many ? rows : (rows + 3) / 4;
    const int weight_groups = p.a.weights_out ? (p.c.max_blocks + 255) / 256 : 0;
    const dim3 grid(row_groups + weight_groups, p.c.kv_heads, p.c.batch);
    if (grid.x == 0) return kStatusOk;
    if (many)
        kv_join_kernel<TYPE, D, 4><<<grid, 256, 0, stream>>>(p, row_groups);
    else
        kv_join_kernel<TYPE, D, 1><<<grid, 256, 0, stream>>>(p, row_groups);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <int TYPE, bool JOIN>
int launch_dim(const KvAttend& p, hipStream_t stream) {
    switch (p.c.head_dim) {
        case 64: return JOIN ? launch_join<TYPE, 64>(p, stream) : launch<TYPE, 64>(p, stream);
        case 128: return JOIN ? launch_join<TYPE, 128>(p, stream) : launch<TYPE, 128>(p, stream);
        case 192: return JOIN ? launch_join<TYPE, 192>(p, stream) : launch<TYPE, 192>(p, stream);
        default: return JOIN ? launch_join<TYPE, 256>(p, stream) : launch<TYPE, 256>(p, stream);
    }
}

template <bool JOIN>
int launch_type(const KvAttend& p, hipStream_t stream) {
    switch (p.a.type) {
        case ROCKNPU_KV_F32: return launch_dim<ROCKNPU_KV_F32, JOIN>(p, stream);
        case ROCKNPU_KV_F16: return launch_dim<ROCKNPU_KV_F16, JOIN>(p, stream);
        default: return launch_dim<ROCKNPU_KV_BF16, JOIN>(p, stream);
    }
}

}  // namespace

int launch_kv_stream(const KvAttend& p, hipStream_t stream) { return launch_type<false>(p, stream); }
int launch_kv_join(const KvAttend& p, hipStream_t stream) { return launch_type<true>(p, stream); }

}  // namespace rk
