// Attention over the 8-bit key/value cache (include/rocknpu_kv.h).
#include <algorithm>
#include <climits>

#include "kv_attend.h"

namespace rk {
namespace {

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
    if ((a->rows > 1 && a->out_row < c->head_dim) || (a->heads > 1 && a->out_head < c->head_dim)) return false;
    if (std::min(a->max_new, a->rows) * (a->heads / c->kv_heads) > INT_MAX) return false;
    if (a->weights_out && (!c->weights || a->max_new * (a->heads / c->kv_heads) > kKvMaxWeightRows)) return false;
    return true;
}

size_t padded(size_t n) { return (n + 255) / 256 * 256; }

// The streaming kernel reads the cache once per tile of 16 rows, the prompt kernel
// once per 128, with several times the work for a block and a longer start.
// Streaming serves calls of at most 32 rows a kv head, and launches of up to four
// tiles and, in tiles times blocks of 128 dims, 100 a CU. 8 kv heads of 128, 4
// heads each, bf16, streaming and prompt kernel: 16 rows x 4 over 4000 tokens 15.0
// and 20.1 us, over 16000 25.6 and 29.5, 32 x 4 over 16000 37.6 and 35.3, 256 x 4
// over 1500 33.5 and 37.5 (110 a CU), 512 x 4 over 2000 75 and 54, two times 512 x
// 4 over 0 39 and 25 (eight tiles a CU). f32: 20 x 4 over 16000 32.2 and 37.0, 12
// x 4 of 8 sequences over 4000 46.7 and 44.5 (94), 512 x 4 over 2000 85 and 66.
constexpr int64_t kStreamRows = 32, kStreamTiles = 4, kStreamWork = 100 * 128;
// Up to this many blocks a workgroup takes them alone; and blocks of a split, at
// least, where they are shared out (8 kv heads of 128, one row, one launch alone
// against splits and their join: 16 blocks 8.4 and 12.7 us, 32 blocks 11.9 and
// 13.1, 48 blocks 15.2 and 13.5; 125 blocks in splits of 8, 16 and 32: 14.9, 16.6
// and 19.2).
constexpr int kAlone = 32;
constexpr int kMinChunk = 8;
// Sequences up to which their blocks are shared out over the workgroups.
constexpr int kMaxShared = 1024;

struct Plan {
    KvAttend p;
    bool stream;
    size_t out_bytes, state_bytes, sums_bytes, slot_bytes;
    size_t bytes() const { return out_bytes + state_bytes + sums_bytes + slot_bytes; }
};

Plan plan(const rocknpu_kv_cache& c, const rocknpu_kv_attention_args& a, int cus) {
    Plan r{};
    KvAttend& p = r.p;
    p.c = c;
    p.a = a;
    p.a.max_new = std::min(a.max_new, a.rows);
    // Below 2^52 such a cap changes a score by less than its last place, and above f32's spacing leaves the softmax the
    // largest alone, capped or not; its reciprocal could fall below f32's range.
    if (a.softcap > 0x1p64f) p.a.softcap = 0.0f;
    p.group = a.heads / c.kv_heads;
    const int64_t per = a.type == ROCKNPU_KV_F32 ? 4 : 8;
    p.vec_q = aligned(a.q, 16) && a.q_row % per == 0 && a.q_head % per == 0;
    p.vec_out = aligned(a.out, 16) && a.out_row % per == 0 && a.out_head % per == 0;
    const int64_t rows = std::max<int64_t>(p.a.max_new, 1) * p.group;
    int64_t blocks = a.max_tokens > 0 ? (a.max_tokens - 1) / kKvBlock + 1 : c.max_blocks;
    if (a.window > 0) blocks = std::min<int64_t>(blocks, (static_cast<int64_t>(a.window) + p.a.max_new) / kKvBlock + 2);
    blocks = std::max<int64_t>(1, std::min<int64_t>(blocks, c.max_blocks));
    const int64_t tiles = (rows + kKvTileRows - 1) / kKvTileRows * c.batch * c.kv_heads;
    r.stream = rows <= kStreamRows || a.weights_out ||
               (tiles <= kStreamTiles * cus && tiles * blocks * c.head_dim <= kStreamWork * cus);
    p.tile_rows = r.stream ? kKvTileRows : kv_prompt_tile();
    p.row_tiles = static_cast<int>((rows + p.tile_rows - 1) / p.tile_rows);
    p.min_chunk = kMinChunk;
    // A streaming workgroup's waves. Eight cut a context into half as many splits and shorten a short one; four even out
    // unequal lengths better where sequences times kv heads come near the CUs (8 kv heads of 128, bf16, in workgroups of
    // eight and of four: one sequence of 16000 tokens 17.7 and 20.3 us, 8 of 1000-3400 19.9 and 20.4, 24 of 600-4000 37.5
    // and 34.5, 32 of 800-3900 40.1 and 36.9; 32 of 4100 each, which the host cannot tell from them, 66 and 77; 4 kv heads
    // of 64, f32, one of 512 7.5 and 7.9, of 900 10.0 and 11.3). Heads of 192 take up to 240 registers: two waves a SIMD,
    // which workgroups of four would not reach; heads of 256 take all of them: one.
    const bool busy = static_cast<int64_t>(c.batch) * c.kv_heads * p.row_tiles >= cus / 2;
    p.waves = c.head_dim == 192 || (c.head_dim <= 128 && !busy) ? 8 : 4;
    // One round of the workgroups that the GPU holds at once: a second round pays every workgroup's start (lookups, the
    // queries, the first blocks' latency) again (32 sequences of 500-4000 tokens, 8 kv heads of 128, workgroups of
    // eight: 44 us; one and a half, two and three rounds 53, 55 and 54). The prompt kernel shares blocks out where that
    // gives every sequence and tile at least four parts: below, joining costs what it saves.
    const int held = !r.stream          ? (c.head_dim <= 128 ? 2 : 1)
                     : c.head_dim == 64 ? (busy ? 3 : 2)
                     : c.head_dim == 128 && busy ? 2 : 1;
    const int64_t resident = static_cast<int64_t>(held) * cus;
    p.whole = static_cast<int>(std::max<int64_t>(
        std::min<int64_t>(resident / (static_cast<int64_t>(c.kv_heads) * p.row_tiles), c.batch * ((blocks + p.min_chunk - 1) / p.min_chunk)), 1));
    const int64_t share = std::max<int64_t>(p.whole - static_cast<int64_t>(c.batch) * (kKvShares - 1) / 4, 1);
    // the device adds up all sequences' blocks in 32 bits
    const bool shared = blocks > (r.stream ? kAlone : kMinChunk) && c.batch <= kMaxShared && rows > 0 &&
                        static_cast<int64_t>(c.batch) * c.max_blocks < (1 << 30);
    p.share = shared && share >= (r.stream ? 2 : 4) ? static_cast<int>(share) : 0;
    for (int k = 0; k < kKvShares; ++k)
        p.per_part[k] = 1.000001f / static_cast<float>(std::max<int64_t>(p.whole - static_cast<int64_t>(c.batch) * k / 4, 1));
    p.slots = p.share + c.batch;
    const size_t slots = static_cast<size_t>(p.slots) * c.kv_heads * p.row_tiles * p.tile_rows;
    if (p.share) r.out_bytes = padded(slots * c.head_dim * 4);
    if (p.share) r.slot_bytes = padded(static_cast<size_t>(c.batch) * sizeof(int2));
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

extern "C" int rocknpu_hip_kv_attention_parts(const rocknpu_kv_cache* cache, const rocknpu_kv_attention_args* args,
                                              int cus, const int32_t* blocks, int32_t* parts, int64_t* slots) {
    using namespace rk;
    if (!blocks || !parts || !slots || !attention_ok(cache, args)) return kStatusInvalid;
    const KvAttend p = plan(*cache, *args, cus > 0 ? cus : device_cu_count()).p;
    *slots = p.slots;
    const auto held = [&](int b) { return std::min(std::max(blocks[b], 0), cache->max_blocks); };
    int64_t all = 0;
    for (int b = 0; b < cache->batch; ++b) all += held(b);
    if (p.share == 0) {
        std::fill(parts, parts + cache->batch, 1);
        return kStatusOk;
    }
    const int chunk = kv_chunk(p, static_cast<int>(all), [&](int c) {
        int n = 0;
        for (int b = 0; b < cache->batch; ++b) n += (held(b) + c - 1) / c;
        return n;
    });
    for (int b = 0; b < cache->batch; ++b) parts[b] = std::min((held(b) + chunk - 1) / chunk, kKvMaxSplits);
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
    uint8_t* at = static_cast<uint8_t*>(workspace);
    if (r.out_bytes) r.p.part_out = reinterpret_cast<float*>(at);
    if (r.state_bytes) r.p.part_state = reinterpret_cast<float*>(at + r.out_bytes);
    if (r.sums_bytes) r.p.block_sums = reinterpret_cast<float*>(at + r.out_bytes + r.state_bytes);
    if (r.slot_bytes) r.p.slots_of = reinterpret_cast<int2*>(at + r.out_bytes + r.state_bytes + r.sums_bytes);
    const int st = r.stream ? launch_kv_stream(r.p, s) : launch_kv_prompt(r.p, s);
    return st == kStatusOk ? launch_kv_join(r.p, s) : st;
}
