// The 8-bit key/value cache (include/rocknpu_kv.h): append, read back, evict.
#include <algorithm>
#include <climits>

#include "kv.h"

namespace rk {
namespace {

constexpr int kAppendThreads = 256;

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    return __float_as_uint(wave_max_nonneg(__uint_as_float(v)));
}

// 16 bytes of elements as f32. `vec`: 16-byte aligned.
template <int TYPE>
__device__ __forceinline__ void load_piece(const typename KvType<TYPE>::T* p, bool vec,
                                           float (&x)[16 / sizeof(typename KvType<TYPE>::T)]) {
    using K = KvType<TYPE>;
    constexpr int kPer = 16 / sizeof(typename K::T);
    if (vec) {
        struct alignas(16) Quad {
            typename K::T e[kPer];
        };
        const Quad v = *reinterpret_cast<const Quad*>(p);
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = K::to_f32(v.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = K::to_f32(p[e]);
    }
}

__device__ __forceinline__ int8_t code_of(float x, float inv) {
    return static_cast<int8_t>(static_cast<int>(fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f)));
}

struct AppendArgs {
    const void *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    const int32_t *past, *cu;
    rocknpu_kv_cache c;
    int rows, max_new;
    bool vec;
};

// One workgroup per touched block of a sequence and head: the new rows, 16 bytes
// a lane, stay in registers while the workgroup finds their largest magnitudes;
// their codes pass through LDS and leave in page order, 16 bytes a lane. Bound by
// the bytes of the rows and codes: 8192 rows of 8 heads of 128, bf16, 50 MB in
// 15.0 us (3.4 TB/s; row by row 29 us); a single token by its chain of lookups, 4.5.
template <int TYPE, int D>
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(AppendArgs a) {
    using T = typename KvType<TYPE>::T;
    constexpr int kPer = 16 / sizeof(T);                          // elements of a piece of a row
    constexpr int kPieces = kKvBlock * D / kPer, kRounds = (kPieces + kAppendThreads - 1) / kAppendThreads;
    constexpr int kChunks = kKvBlock * D / 16;                    // 16-byte pieces of a page's keys, and of its values
    __shared__ uint32_t red[2][kAppendThreads / 64];
    __shared__ alignas(16) int8_t codes[2][kKvBlock][D + 4];
    const int tid = threadIdx.x, b = blockIdx.z, h = blockIdx.y;
    int gone;
    const KvSpan s = kv_span(a.past, a.cu, a.c.dropped, b, a.rows, a.max_new, gone);
    const int j = s.past / kKvBlock + blockIdx.x;
    const int lead = max(s.past - j * kKvBlock, 0);          // tokens the block held before
    const int end = min(s.past + s.n - j * kKvBlock, kKvBlock);
    if (end <= lead) return;
    const int64_t row = s.row0 + (j * kKvBlock - s.past);     // the row of the block's token 0

    // the rows' loads go out before the table's, which they do not wait for
    float x[2][kRounds][kPer];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const T* src = static_cast<const T*>(w ? a.v : a.k) + h * (w ? a.v_head : a.k_head);
        const int64_t stride = w ? a.v_row : a.k_row;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = tid + r * kAppendThreads, t = i / (D / kPer);
            if (t >= lead && t < end) {
                load_piece<TYPE>(src + (row + t) * stride + i % (D / kPer) * kPer, a.vec, x[w][r]);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) x[w][r][e] = 0.0f;
            }
        }
    }
    const int64_t entry_row = (static_cast<int64_t>(b) * a.c.kv_heads + h) * a.c.max_blocks;
    const int at = j - gone;
    if (at < 0 || at >= a.c.max_blocks) return;
    const int page = a.c.table[entry_row + at];
    if (page < 0 || page >= a.c.n_pages) return;
    int8_t* keys = reinterpret_cast<int8_t*>(a.c.pages) + static_cast<int64_t>(page) * (2 * kKvBlock * D);
    float before[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) before[w] = lead > 0 ? a.c.scales[2 * static_cast<int64_t>(page) + w] : 0.0f;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t top = 0;
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
#pragma unroll
            for (int e = 0; e < kPer; ++e) top = max(top, __float_as_uint(x[w][r][e]) & 0x7fffffffu);
        top = wave_max_u32(top);
        if ((tid & 63) == 0) red[w][tid >> 6] = top;
    }
    __syncthreads();
    float again[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t top = red[w][0];
#pragma unroll
        for (int i = 1; i < kAppendThreads / 64; ++i) top = max(top, red[w][i]);
        // bit patterns above FLT_MAX are infinities and NaNs; so is a scale below 0 to the readers
        const bool bad = top > 0x7f7fffffu || !(before[w] >= 0.0f && before[w] <= 3.402823466e38f);
        const float scale = bad ? __builtin_nanf("") : fmaxf(fmaxf(__uint_as_float(top) / 127.0f, before[w]), kKvScaleFloor);
        const float inv = bad ? 0.0f : 1.0f / scale;
        again[w] = bad ? 0.0f : before[w] / scale;
        // all threads read the scales before the barrier above
        if (tid == 0) a.c.scales[2 * static_cast<int64_t>(page) + w] = scale;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = tid + r * kAppendThreads, t = i / (D / kPer);
            if (t < kKvBlock) {
                uint32_t* to = reinterpret_cast<uint32_t*>(&codes[w][t][i % (D / kPer) * kPer]);
#pragma unroll
                for (int e = 0; e < kPer / 4; ++e) {
                    uint32_t q = 0;
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        q |= bad ? 0u : static_cast<uint32_t>(code_of(x[w][r][e * 4 + f], inv) & 0xff) << (8 * f);
                    to[e] = q;
                }
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < kChunks; i += kAppendThreads) {
        // keys: token i / 4 % 32, dims 64 (i / 128) + 16 (i % 4)
        const int t = i / 4 % kKvBlock;
        if (t >= lead && t < end) {
            const uint32_t* row_lds = reinterpret_cast<const uint32_t*>(&codes[0][t][i / 128 * 64 + i % 4 * 16]);
            *reinterpret_cast<uint4*>(keys + i * 16) = make_uint4(row_lds[0], row_lds[1], row_lds[2], row_lds[3]);
        } else if (t < lead && again[0] != 1.0f) {
            alignas(16) int8_t q[16];
            *reinterpret_cast<uint4*>(q) = *reinterpret_cast<uint4*>(keys + i * 16);
#pragma unroll
            for (int e = 0; e < 16; ++e) q[e] = code_of(static_cast<float>(q[e]), again[0]);
            *reinterpret_cast<uint4*>(keys + i * 16) = *reinterpret_cast<uint4*>(q);
        }
        // values: 8 tokens of dims d and d + 16
        const int d = i / 64 * 32 + i / 4 % 16, t4 = i % 4 * 4;
        int8_t* values = keys + kKvBlock * D + i * 16;
        alignas(16) int8_t q[16];
        if (lead > 0) *reinterpret_cast<uint4*>(q) = *reinterpret_cast<uint4*>(values);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int tv = e / 4 % 2 * 16 + t4 + e % 4;
            if (tv < lead)
                q[e] = code_of(static_cast<float>(q[e]), again[1]);
            else
                q[e] = codes[1][tv][d + e / 8 * 16];
        }
        *reinterpret_cast<uint4*>(values) = *reinterpret_cast<uint4*>(q);
    }
    if (tid == 0 && lead == 0) {
        a.c.starts[entry_row + at] = j * kKvBlock;
        if (a.c.weights) a.c.weights[entry_row + at] = 0.0f;
    }
}

// Place of the block that starts at `start` among a row's `n` ascending starts,
// or -1.
__device__ __forceinline__ int find_block(const int32_t* starts, int n, int start) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] < start)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo < n && starts[lo] == start ? lo : -1;
}

// One workgroup per block of a sequence and head that holds a position asked for,
// through LDS, so that both the page and the rows are whole runs of 16 bytes a
// lane. Bound by the bytes of codes and rows: 8192 positions of 8 heads of 128,
// bf16, 50 MB in 10.6 us (4.7 TB/s, a large copy's rate).
template <int TYPE, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(rocknpu_kv_cache c, const int32_t* __restrict__ first,
                                                      const int32_t* __restrict__ tokens, int64_t count,
                                                      typename KvType<TYPE>::T* __restrict__ k,
                                                      typename KvType<TYPE>::T* __restrict__ v) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    constexpr int kChunks = kKvBlock * D / 16;
    __shared__ alignas(16) int8_t codes[2][kKvBlock][D + 4];
    const int tid = threadIdx.x, b = blockIdx.z, h = blockIdx.y;
    const int total = min(max(tokens[b], 0), 0x3fffffff);
    const int gone = max(c.dropped[b], 0);
    const int held = min((total + kKvBlock - 1) / kKvBlock - gone, c.max_blocks);
    const int64_t entry_row = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks;
    const int64_t from = first[b];
    const int64_t start = ((from - (from < 0 ? kKvBlock - 1 : 0)) / kKvBlock + blockIdx.x) * kKvBlock;
    if (start >= from + count) return;
    int page = -1;
    if (start >= 0 && start < total) {
        int at = static_cast<int>(start / kKvBlock);
        if (gone) at = find_block(c.starts + entry_row, held, static_cast<int>(start));
        page = at >= 0 && at < held ? c.table[entry_row + at] : -1;
        if (page >= c.n_pages) page = -1;
    }
    const int8_t* keys = reinterpret_cast<const int8_t*>(c.pages) + static_cast<int64_t>(max(page, 0)) * (2 * kKvBlock * D);
    const float2 scale = reinterpret_cast<const float2*>(c.scales)[max(page, 0)];
    constexpr int kRounds = (kChunks + 255) / 256, kPer = 16 / sizeof(T);
    struct alignas(16) Quad {
        T e[kPer];
    };
    uint4 key[kRounds] = {}, value[kRounds] = {};
    if (page >= 0) {
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = tid + r * 256;
            if (i < kChunks) {
                key[r] = *reinterpret_cast<const uint4*>(keys + i * 16);
                value[r] = *reinterpret_cast<const uint4*>(keys + kKvBlock * D + i * 16);
            }
        }
    }
    // keys: token i / 4 % 32, dims 64 (i / 128) + 16 (i % 4); values: 8 tokens of dims d and d + 16
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int i = tid + r * 256;
        if (i < kChunks) {
            uint32_t* row = reinterpret_cast<uint32_t*>(&codes[0][i / 4 % kKvBlock][i / 128 * 64 + i % 4 * 16]);
            row[0] = key[r].x;
            row[1] = key[r].y;
            row[2] = key[r].z;
            row[3] = key[r].w;
            const int d = i / 64 * 32 + i / 4 % 16, t4 = i % 4 * 4;
            const int8_t* q = reinterpret_cast<const int8_t*>(&value[r]);
#pragma unroll
            for (int e = 0; e < 16; ++e) codes[1][e / 4 % 2 * 16 + t4 + e % 4][d + e / 8 * 16] = q[e];
        }
    }
    __syncthreads();
    // 16 bytes of a row a thread
    for (int i = tid; i < 2 * kKvBlock * D / kPer; i += 256) {
        const int w = i / (kKvBlock * D / kPer), t = i / (D / kPer) % kKvBlock, d = i % (D / kPer) * kPer;
        const int64_t o = start + t - from;
        if (o < 0 || o >= count) continue;
        const bool there = page >= 0 && start + t < total;
        Quad quad;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            float x = static_cast<float>(codes[w][t][d + e]) * (w ? scale.y : scale.x);
            // the f32 product is the value: not joined with the conversion to f16, which would round it once only
            asm("" : "+v"(x));
            quad.e[e] = K::from_f32(there ? x : 0.0f);
        }
        *reinterpret_cast<Quad*>((w ? v : k) + ((static_cast<int64_t>(b) * count + o) * c.kv_heads + h) * D + d) = quad;
    }
}

// An order-preserving map of weights to whole numbers: NaN is 0, -0 equals +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of `v` over the threads before this one.
template <int THREADS>
__device__ __forceinline__ int exclusive_sum(int v, int* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int x = wave_scan(v);
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) before += w < wave ? part[w] : 0;
    return before + x - v;
}

// One workgroup per row of the table, entry i * THREADS + thread in register i of
// a thread. The budget-th greatest key is found by digits of 11, 11 and 10 bits
// from the top (a histogram in LDS of the entries that match the digits found so
// far): the first digit holds the exponent and two more bits, so that few of a
// wave's lanes meet in one bin (with digits of 8 bits 512 rows of 4098 took 10 us
// more). The histograms are cleared while the row's loads are in flight, and sums
// over threads run through DPP (15 us; cleared pass by pass and by __shfl 20, of
// which 50 MB take 11 at a large copy's rate). Then ballots and one sum over (register, wave) place every
// entry. Everything is read before the first write, so outputs may be the inputs.
// Bound by the latency of its steps where rows are few, else by its bytes.
template <int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void kv_evict_kernel(rocknpu_kv_evict_args a) {
    constexpr int kWaves = THREADS / 64, kBins = 2048, kGroups = ITEMS * kWaves;
    static_assert(kGroups <= THREADS);
    __shared__ int hists[3][kBins];
    __shared__ int part[kWaves];
    __shared__ int pick[2];                   // the digit found, and how many entries rank above it
    __shared__ int count[kGroups][2];         // by register and wave: entries above the key found, and equal to it
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const int b = static_cast<int>(r / a.kv_heads);
    const int64_t base = r * a.max_blocks;
    int32_t page[ITEMS], start[ITEMS];
    float w[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int at = min(i * THREADS + tid, a.max_blocks - 1);
        w[i] = a.weights[base + at];
        page[i] = a.table[base + at];
        start[i] = a.starts[base + at];
    }
    const int total = min(max(a.tokens[b], 0), 0x3fffffff);
    const int gone = max(a.dropped[b], 0);
    for (int i = tid; i < 3 * kBins; i += THREADS) hists[0][i] = 0;
    __syncthreads();
    const int n = min(max((total + kKvBlock - 1) / kKvBlock - gone, 0), a.max_blocks);
    uint32_t key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int at = i * THREADS + tid;
        key[i] = at < a.sinks || at >= n - a.recent ? 0xffffffffu : weight_key(w[i]);
    }
    int to[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) to[i] = i * THREADS + tid;
    if (n > a.budget) {
        uint32_t found = 0;
        int above = 0;  // entries known to rank above the budget-th
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
            int* hist = hists[pass];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (i * THREADS + tid < n && (pass == 0 || key[i] >> (pass == 1 ? 21 : 10) == found))
                    atomicAdd(&hist[key[i] >> shift & (bins - 1)], 1);
            __syncthreads();
            // this thread's bins, from the top
            constexpr int kMost = kBins / THREADS > 0 ? kBins / THREADS : 1;
            const int mine = bins / THREADS > 0 ? bins / THREADS : 1;
            int c[kMost], sum = 0;
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                c[i] = i < mine && tid * mine + i < bins ? hist[bins - 1 - tid * mine - i] : 0;
                sum += c[i];
            }
            int up = above + exclusive_sum<THREADS>(sum, part);
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                if (up < a.budget && up + c[i] >= a.budget) {
                    pick[0] = bins - 1 - tid * mine - i;
                    pick[1] = up;
                }
                up += c[i];
            }
            __syncthreads();
            found = found << (pass == 2 ? 10 : 11) | static_cast<uint32_t>(pick[0]);
            above = pick[1];
        }
        // Of the entries equal to the budget-th key the first `need` stay: an entry has as many kept ones before it as there
        // are above the key, and equal to it but no more than `need`.
        const int need = a.budget - above;
        uint64_t over[ITEMS], same[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool in = i * THREADS + tid < n;
            over[i] = __ballot(in && key[i] > found);
            same[i] = __ballot(in && key[i] == found);
            if (lane == 0) {
                count[i * kWaves + wave][0] = __popcll(over[i]);
                count[i * kWaves + wave][1] = __popcll(same[i]);
            }
        }
        __syncthreads();
        // both sums in one number: neither reaches 2^16
        const int packed = tid < kGroups ? count[tid][0] << 16 | count[tid][1] : 0;
        const int before = exclusive_sum<THREADS>(packed, part);
        if (tid < kGroups) {
            count[tid][0] = before >> 16;
            count[tid][1] = before & 0xffff;
        }
        __syncthreads();
        const uint64_t lower = (uint64_t{1} << lane) - 1;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = i * THREADS + tid;
            const int equal = count[i * kWaves + wave][1] + __popcll(same[i] & lower);
            const int kept = count[i * kWaves + wave][0] + __popcll(over[i] & lower) + min(equal, need);
            const bool keep = (over[i] >> lane & 1) || ((same[i] >> lane & 1) && equal < need);
            if (at < n) to[i] = keep ? kept : a.budget + at - kept;
        }
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (i * THREADS + tid >= a.max_blocks) break;
        a.table_out[base + to[i]] = page[i];
        a.starts_out[base + to[i]] = start[i];
        a.weights_out[base + to[i]] = w[i];
    }
    if (tid == 0 && r % a.kv_heads == 0) a.dropped_out[b] = a.dropped[b] + max(n - a.budget, 0);
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int element_size(uint32_t type) { return type == ROCKNPU_KV_F32 ? 4 : 2; }

template <int TYPE>
void launch_append(const AppendArgs& a, dim3 grid, hipStream_t s) {
    switch (a.c.head_dim) {
        case 64: kv_append_kernel<TYPE, 64><<<grid, kAppendThreads, 0, s>>>(a); break;
        case 128: kv_append_kernel<TYPE, 128><<<grid, kAppendThreads, 0, s>>>(a); break;
        case 192: kv_append_kernel<TYPE, 192><<<grid, kAppendThreads, 0, s>>>(a); break;
        default: kv_append_kernel<TYPE, 256><<<grid, kAppendThreads, 0, s>>>(a); break;
    }
}

template <int TYPE>
void launch_read(const rocknpu_kv_cache& c, const int32_t* first, const int32_t* tokens, int64_t count, void* k, void* v,
                 hipStream_t s) {
    using T = typename KvType<TYPE>::T;
    // a run of `count` positions touches at most this many blocks, wherever in a block it begins
    const dim3 grid(static_cast<unsigned>((count + 2 * kKvBlock - 2) / kKvBlock), c.kv_heads, c.batch);
    T *kt = static_cast<T*>(k), *vt = static_cast<T*>(v);
    switch (c.head_dim) {
        case 64: kv_read_kernel<TYPE, 64><<<grid, 256, 0, s>>>(c, first, tokens, count, kt, vt); break;
        case 128: kv_read_kernel<TYPE, 128><<<grid, 256, 0, s>>>(c, first, tokens, count, kt, vt); break;
        case 192: kv_read_kernel<TYPE, 192><<<grid, 256, 0, s>>>(c, first, tokens, count, kt, vt); break;
        default: kv_read_kernel<TYPE, 256><<<grid, 256, 0, s>>>(c, first, tokens, count, kt, vt); break;
    }
}

int status() { return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec; }

}  // namespace

bool kv_cache_ok(const rocknpu_kv_cache* c) {
    if (!c || !c->pages || !c->scales || !c->table || !c->starts || !c->dropped) return false;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 192 && c->head_dim != 256) return false;
    if (c->n_pages < 1 || c->n_pages > INT_MAX || c->batch < 1 || c->batch > kKvMaxBatch || c->kv_heads < 1 ||
        c->kv_heads > 65535 || c->max_blocks < 1 || c->max_blocks > INT_MAX / kKvBlock)
        return false;
    return aligned(c->pages, 16) && aligned(c->scales, 8) && aligned(c->table, 4) && aligned(c->starts, 4) &&
           aligned(c->dropped, 4) && aligned(c->weights, 4);
}

}  // namespace rk

extern "C" int rocknpu_hip_kv_append(const rocknpu_kv_cache* cache, uint32_t type, const void* k, int64_t k_row,
                                     int64_t k_head, const void* v, int64_t v_row, int64_t v_head, size_t rows,
                                     const int32_t* past, const int32_t* cu, size_t max_new, void* stream) {
    using namespace rk;
    if (!kv_cache_ok(cache) || type > ROCKNPU_KV_BF16 || !past || !cu || rows > INT_MAX || max_new > INT_MAX)
        return kStatusInvalid;
    if (rows == 0 || max_new == 0) return kStatusOk;
    if (!k || !v || k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0) return kStatusInvalid;
    const int size = element_size(type);
    if (!aligned(k, size) || !aligned(v, size)) return kStatusInvalid;
    max_new = std::min(max_new, rows);
    AppendArgs a{k, v, k_row, k_head, v_row, v_head, past, cu, *cache, static_cast<int>(rows), static_cast<int>(max_new), false};
    const int64_t per = 16 / size;
    a.vec = aligned(k, 16) && aligned(v, 16) && k_row % per == 0 && k_head % per == 0 && v_row % per == 0 && v_head % per == 0;
    // a sequence's rows touch at most this many blocks, wherever in a block they begin
    const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(max_new) + 2 * kKvBlock - 2) / kKvBlock);
    const dim3 grid(blocks, cache->kv_heads, cache->batch);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == ROCKNPU_KV_F32)
        launch_append<ROCKNPU_KV_F32>(a, grid, s);
    else if (type == ROCKNPU_KV_F16)
        launch_append<ROCKNPU_KV_F16>(a, grid, s);
    else
        launch_append<ROCKNPU_KV_BF16>(a, grid, s);
    return status();
}

extern "C" int rocknpu_hip_kv_read(const rocknpu_kv_cache* cache, const int32_t* first, const int32_t* tokens,
                                   size_t count, uint32_t type, void* k, void* v, void* stream) {
    using namespace rk;
    if (!kv_cache_ok(cache) || type > ROCKNPU_KV_BF16 || !first || !tokens || count > INT_MAX) return kStatusInvalid;
    if (count == 0) return kStatusOk;
    if (!k || !v || !aligned(k, 16) || !aligned(v, 16)) return kStatusInvalid;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t n = static_cast<int64_t>(count);
    if (type == ROCKNPU_KV_F32)
        launch_read<ROCKNPU_KV_F32>(*cache, first, tokens, n, k, v, s);
    else if (type == ROCKNPU_KV_F16)
        launch_read<ROCKNPU_KV_F16>(*cache, first, tokens, n, k, v, s);
    else
        launch_read<ROCKNPU_KV_BF16>(*cache, first, tokens, n, k, v, s);
    return status();
}

extern "C" int rocknpu_hip_kv_evict(const rocknpu_kv_evict_args* args, void* stream) {
    using namespace rk;
    if (!args) return kStatusInvalid;
    const rocknpu_kv_evict_args& a = *args;
    if (!a.table || !a.starts || !a.weights || !a.tokens || !a.dropped || !a.table_out || !a.starts_out ||
        !a.weights_out || !a.dropped_out || a.dropped_out == a.dropped)
        return kStatusInvalid;
    if (a.batch < 1 || a.kv_heads < 1 || a.max_blocks < 1 || a.max_blocks > kKvEvictMaxBlocks || a.sinks < 0 ||
        a.recent < 1 || a.budget < 1 || static_cast<int64_t>(a.sinks) + a.recent > a.budget ||
        static_cast<int64_t>(a.batch) * a.kv_heads > INT_MAX)
        return kStatusInvalid;
    const dim3 grid(static_cast<unsigned>(a.batch * a.kv_heads));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.max_blocks <= 256)
        kv_evict_kernel<256, 1><<<grid, 256, 0, s>>>(a);
    else if (a.max_blocks <= 1024)
        kv_evict_kernel<256, 4><<<grid, 256, 0, s>>>(a);
    else if (a.max_blocks <= 4096)
        kv_evict_kernel<1024, 4><<<grid, 1024, 0, s>>>(a);
    else
        kv_evict_kernel<1024, 16><<<grid, 1024, 0, s>>>(a);
    return status();
}
