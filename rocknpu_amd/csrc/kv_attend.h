// What the attention kernels over the 8-bit key/value cache share: a launch's
// description, the range of blocks that rows see, and code conversions.
//
// Softmax over blocks with scales of their own. With keys kc * sk and values
// vc * sv in a block (kc, vc whole numbers), and everything in powers of two,
//   o = sum 2^y vc / sum 2^y / sv,   y = x log2(e) + log2(sv) - M
// for any M: folding a block's value scale into the exponent leaves the codes
// as they are (exact in f16 and bf16), takes one add per block and row, and one
// product per block and row for the denominator. M is the row's running maximum
// of x log2(e) + log2(sv). A scale below kKvFoldLeast (blocks of zeros have
// 2^-100) counts as kKvFoldLeast in M, and its block's denominator is summed apart
// with that one: with its own, the keys' share would fall below f32's range where
// other blocks' values are large, and pass it where it is divided by the scale.
#pragma once

#include "kv.h"

namespace rk {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kKvMaxSplits = 256;  // workgroups that share a tile's blocks, at most
constexpr int kKvShares = 4;       // lengths of a split that are tried
constexpr int kKvTileRows = 16;  // rows of a tile of the streaming kernel

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

struct KvAttend {
    rocknpu_kv_cache c;
    rocknpu_kv_attention_args a;
    int group;       // heads per kv head
    int row_tiles;   // tiles of rows that a sequence and kv head may have
    int tile_rows;
    int waves;       // of a streaming workgroup
    // per kv head and row tile:
    int share;       // parts that all sequences' blocks are cut into at least; 0: one workgroup each
    int slots;       // workgroups: share + batch, or batch
    int whole;       // workgroups that the GPU holds at once, or as many as there can be work for; at most slots
    float per_part[kKvShares];  // 1 / parts, rounded up, in the order in which they are tried; the last is share
    int min_chunk;   // blocks per workgroup, at least
    bool vec_q, vec_out;
    // workspace, one entry per (kv head, row tile, slot): sums of the output [rows][head_dim], maxima and sums
    // [rows][2]; one per (sequence, kv head, block, row): its weight's sum and the maximum it refers to
    float* part_out;
    float* part_state;
    float* block_sums;
    int2* slots_of;  // a sequence's first slot and how many it has
};

// A page's scale, NaN where there is none or it is negative or not finite.
__device__ __forceinline__ float kv_scale(float s, bool ok) {
    return ok && s >= 0.0f && s <= 3.402823466e38f ? s : __builtin_nanf("");
}

// Whether the exponents of a block's weights take its value scale as it is (NaN
// is): the same in every lane.
constexpr float kKvFoldLeast = 0x1p-40f;
__device__ __forceinline__ bool kv_folds(float sv) { return !(sv < kKvFoldLeast); }

// How many of a row's n ascending starts are below `value`: 64 probes a round,
// the same answer in every lane.
__device__ __forceinline__ int starts_below(const int32_t* starts, int n, int value) {
    const int lane = threadIdx.x & 63;
    int lo = 0, size = n;  // the count lies in [lo, lo + size]
    while (size > 0) {
        const int step = (size + 63) / 64;
        const int at = lane * step;
        const bool below = at < size && starts[lo + at] < value;
        const int c = __popcll(__ballot(below));
        if (c == 0) return lo;
        // entry (c - 1) step is below, entry c step (if any) is not
        lo += (c - 1) * step + 1;
        size = min(step - 1, size - (c - 1) * step - 1);
    }
    return lo;
}

// The positions before this one are seen whatever the window; held to a range in
// which sums of positions and sizes stay within 32 bits, as `past` is.
__device__ __forceinline__ int kv_prefix(const rocknpu_kv_attention_args& a, int b) {
    return a.prefix ? min(max(a.prefix[b], 0), 0x3fffffff) : 0;
}

// The blocks that rows at positions q0 .. q1 see: entries [0, first) and
// [from, to) of the table's row.
struct KvRange {
    int first, from, to;
    __device__ __forceinline__ int count() const { return first + to - from; }
    __device__ __forceinline__ int entry(int i) const { return i < first ? i : i - first + from; }
};
__device__ __forceinline__ KvRange kv_range(const rocknpu_kv_attention_args& a, const int32_t* starts, int held, int gone,
                                            int q0, int q1, int prefix) {
    KvRange r{0, 0, max(held, 0)};
    if (!a.causal || held <= 0) return r;
    // newest blocks begin behind the rows
    const int last = max(q1, prefix - 1);
    r.to = min(held, max(last / kKvBlock + 1 - gone, 0));
    if (gone && last / kKvBlock + 1 - gone < held) r.to = starts_below(starts, held, last + 1);
    r.to = uniform(r.to);
    if (a.window == 0) return r;
    const int lowest = q0 - a.window + 1;  // first position that a row's window holds
    if (lowest <= 0) return r;
    const int from_start = lowest / kKvBlock * kKvBlock;
    r.from = min(gone ? starts_below(starts, held, from_start) : from_start / kKvBlock, r.to);
    r.from = uniform(r.from);
    if (prefix > 0) r.first = uniform(min(gone ? starts_below(starts, held, prefix) : (prefix + kKvBlock - 1) / kKvBlock, r.from));
    return r;
}

// Which sequence a slot works on, and which of the sequence's `splits` parts it
// takes (seq < 0: none). Every sequence with rows gets one slot for each `chunk`
// blocks that its rows may see: a batch of unequal lengths loads the GPU evenly.
// Each sequence's last slot may be short, so chunk = all / whole can come to whole
// + batch slots, and what the GPU does not hold at once waits for a round of its
// own; chunks for whole, whole - batch / 4, ... parts are tried until the slots
// fit (17 sequences of 700-15200 tokens, 8 kv heads of 128: 59 us, 75 with whole
// - batch / 2 alone). All workgroups of a launch work out the same division,
// before their first load of the cache: sums over lanes run through DPP and
// quotients through the reciprocal (by __shfl and division it cost one sequence of
// 4000 tokens 1 us of 14).
struct KvSlot {
    int seq, split, splits, first;
};
__device__ __forceinline__ int kv_blocks_estimate(const KvAttend& p, int b) {
    int gone;
    const KvSpan s = kv_span(p.a.past, p.a.cu, p.c.dropped, b, static_cast<int>(p.a.rows), static_cast<int>(p.a.max_new), gone);
    if (s.n == 0) return 0;
    int blocks = min((s.past + s.n + kKvBlock - 1) / kKvBlock - gone, p.c.max_blocks);
    if (p.a.window > 0) {
        const int prefix = kv_prefix(p.a, b);
        blocks = min(blocks, min(p.a.window, 0x3fffffff) / kKvBlock + (s.n + prefix) / kKvBlock + 3);
    }
    return max(blocks, 1);
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
// x / y for whole numbers of which the quotient is below 2^20 (a batch has at most
// kKvShares times as many slots as the GPU holds): by the reciprocal it is off by
// less than one, which is mended.
__device__ __forceinline__ int kv_divide(int x, int y) {
    int q = static_cast<int>(static_cast<float>(x) * __builtin_amdgcn_rcpf(static_cast<float>(y)));
    q -= q * y > x;
    return q + ((q + 1) * y <= x);
}
// Blocks of a split, where all sequences' rows may see `all` blocks together;
// `needed` gives the slots that a chunk comes to. The last chunk fits `slots`
// whatever the sequences' lengths are; a longer one may take more and has to be
// counted. That is done for up to 64 sequences, one a lane: more of them take the
// last chunk (counting 200 of 500-4000 tokens, 2 kv heads of 128, for the longer
// ones too: 65 us, 62 so; 96 of 8 kv heads of 64: 51 and 49). The host asks the
// same function how a call is shared out.
template <class Needed>
__host__ __device__ __forceinline__ int kv_chunk(const KvAttend& p, int all, const Needed& needed) {
    int chunk = 0;
#pragma unroll
    for (int k = 0; k < kKvShares; ++k) {
        if (p.c.batch > 64 && k < kKvShares - 1) continue;
        // at least all / parts: the factor and the 1 outdo the rounding
        chunk = static_cast<int>(static_cast<float>(all) * p.per_part[k]) + 1;
        chunk = chunk > p.min_chunk ? chunk : p.min_chunk;
        if (k == kKvShares - 1 || p.c.batch == 1) break;
        if (needed(chunk) <= p.whole) break;
    }
    return chunk;
}
__device__ __forceinline__ KvSlot kv_slot(const KvAttend& p, int want) {
    const int lane = threadIdx.x & 63, batch = p.c.batch;
    if (p.share == 0) return KvSlot{want, 0, 1, want};
    const int mine = lane < batch ? kv_blocks_estimate(p, lane) : 0;
    int all = mine;
    for (int base = 64; base < batch; base += 64) all += base + lane < batch ? kv_blocks_estimate(p, base + lane) : 0;
    all = wave_sum(all);
    const int chunk = kv_chunk(p, all, [&](int c) { return wave_sum(kv_divide(mine + c - 1, c)); });
    int before = 0;
    for (int base = 0; base < batch; base += 64) {
        const int blocks = base == 0 ? mine : base + lane < batch ? kv_blocks_estimate(p, base + lane) : 0;
        const int splits = min(kv_divide(blocks + chunk - 1, chunk), kKvMaxSplits);
        const int upto = before + wave_scan(splits);
        const unsigned long long hit = __ballot(want < upto);
        if (hit) {
            const int l = uniform(__ffsll(hit) - 1);
            const int end = __builtin_amdgcn_readlane(upto, l), n = __builtin_amdgcn_readlane(splits, l);
            return KvSlot{base + l, want - (end - n), n, end - n};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return KvSlot{-1, 0, 0, 0};
}
// A sequence's slots, for the join: written by one workgroup of its first slot.
__device__ __forceinline__ void kv_leave_slot(const KvAttend& p, const KvSlot& s, int h, int tile) {
    if (p.share && s.split == 0 && h == 0 && tile == 0 && threadIdx.x == 0) p.slots_of[s.seq] = make_int2(s.first, s.splits);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// cap tanh(x / cap), to a few units of the last place however small x / cap is.
// 16-bit calls take tanh z as a quotient: of its continued fraction's fifth
// convergent, z (945 + 105 z^2 + z^4) / (945 + 420 z^2 + 15 z^4), up to 1, and
// (e^2z - 1) / (e^2z + 1) above, which for small z would leave 2^-24 of the cap.
// (8 sequences of 4 rows under a window of 4096 tokens, f16: 23.5 us; by
// 1 - 2 / (1 + e^2z) throughout 23.1.)
template <bool EXACT>
__device__ __forceinline__ float kv_cap(float x, float cap) {
    if constexpr (EXACT) return cap * tanhf(x / cap);
    const float z = x * __builtin_amdgcn_rcpf(cap), z2 = z * z;
    const float e = exp2_fast(2.0f * kLog2e * fminf(fmaxf(z, -20.0f), 20.0f));
    const bool large = fabsf(z) > 1.0f;  // not NaN
    const float over = large ? e - 1.0f : z * __builtin_fmaf(z2, z2 + 105.0f, 945.0f);
    const float under = large ? e + 1.0f : __builtin_fmaf(z2, __builtin_fmaf(15.0f, z2, 420.0f), 945.0f);
    return cap * (over * __builtin_amdgcn_rcpf(under));
}

// Whether a row at qpos sees the key at kpos.
__device__ __forceinline__ bool kv_seen(const rocknpu_kv_attention_args& a, int kpos, int qpos, int prefix, int total) {
    const bool seen = !a.causal || (kpos <= qpos && (a.window == 0 || kpos > qpos - a.window)) || kpos < prefix;
    return seen && kpos < total;
}

// Whether every row at q0 .. q1 sees all of the block that begins at `start`.
__device__ __forceinline__ bool kv_all_seen(const rocknpu_kv_attention_args& a, int start, int q0, int q1, int prefix, int total) {
    const bool seen = !a.causal || (start + kKvBlock - 1 <= q0 && (a.window == 0 || start > q1 - a.window)) ||
                      start + kKvBlock <= prefix;
    return seen && start + kKvBlock <= total;
}

// Eight signed bytes as f16, exactly: byte + 128 lands in the low mantissa bits
// of 1024 (f16 0x6400 + u is 1024 + u), and 1152 comes off again.
__device__ __forceinline__ half8 codes_to_half(uint32_t lo, uint32_t hi) {
    union {
        uint32_t u[4];
        half2v h[4];
        half8 v;
    } r;
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
    const half2v off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
#pragma unroll
    for (int i = 0; i < 4; ++i) r.h[i] = r.h[i] - off;
    return r.v;
}

// Eight signed bytes as bf16, exactly (|code| <= 127 fits its 8 bits): the high
// halves of their f32.
__device__ __forceinline__ bhalf8 codes_to_bhalf(uint32_t lo, uint32_t hi) {
    union {
        uint32_t u[4];
        bhalf8 v;
    } r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? lo : hi;
        const float a = static_cast<float>(static_cast<int8_t>(w >> (i % 2 * 16)));
        const float b = static_cast<float>(static_cast<int8_t>(w >> (i % 2 * 16 + 8)));
        r.u[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    return r.v;
}

// x as the sum of PARTS bf16, eight at a time, each part what the ones before it
// leave, rounded to nearest: 17 bits in two (an error of 2^-18 at most), f32's 24
// in three, over f32's whole range. (Cut off, which costs as much, two hold 16 bits
// and leave outputs closer to 0 by 2^-17 in the mean.)
template <int PARTS>
__device__ __forceinline__ void split_bhalf(const float (&x)[8], bhalf8 (&part)[PARTS]) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        union {
            uint32_t u[4];
            bhalf2v h[4];
            bhalf8 v;
        } r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.h[i] = __builtin_convertvector((float2v{rest[2 * i], rest[2 * i + 1]}), bhalf2v);
        part[p] = r.v;
        if (p + 1 < PARTS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                rest[2 * i] -= __uint_as_float(r.u[i] << 16);
                rest[2 * i + 1] -= __uint_as_float(r.u[i] & 0xffff0000u);
            }
        }
    }
}

// Eight consecutive elements of a row as f32.
template <int TYPE>
__device__ __forceinline__ void load8(const typename KvType<TYPE>::T* p, bool vec, float (&x)[8]) {
    using K = KvType<TYPE>;
    if (vec) {
        constexpr int kPer = 16 / sizeof(typename K::T);
        struct alignas(16) Quad {
            typename K::T e[kPer];
        };
#pragma unroll
        for (int i = 0; i < 8 / kPer; ++i) {
            const Quad v = reinterpret_cast<const Quad*>(p)[i];
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[i * kPer + j] = K::to_f32(v.e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = K::to_f32(p[i]);
    }
}

// The power of two that brings a row of magnitude `top` to 2^13 .. 2^14, where
// f16 holds it with room on both sides (1 for an empty or not finite row).
__device__ __forceinline__ float row_power(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    if (e == -127 || e == 128) return 1.0f;
    return __uint_as_float(static_cast<uint32_t>(127 + min(max(13 - e, -114), 120)) << 23);
}

// kv_stream.hip: tiles of kKvTileRows rows; kv_prompt.hip: of kv_prompt_tile rows.
int launch_kv_stream(const KvAttend& p, hipStream_t stream);
int kv_prompt_tile();
int launch_kv_prompt(const KvAttend& p, hipStream_t stream);
// Joins the parts that either left, and the block weights. kv_stream.hip.
int launch_kv_join(const KvAttend& p, hipStream_t stream);

}  // namespace rk
