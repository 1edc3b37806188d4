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

// 16 consecutive elements as f32. `vec`: 16-byte aligned.
template <int TYPE>
__device__ __forceinline__ void load16(const typename KvType<TYPE>::T* p, bool vec, float (&x)[16]) {
    using K = KvType<TYPE>;
    if (vec) {
        constexpr int kPer = 16 / sizeof(typename K::T);
        struct alignas(16) Quad {
            typename K::T e[kPer];
        };
#pragma unroll
        for (int i = 0; i < 16 / kPer; ++i) {
            const Quad v = reinterpret_cast<const Quad*>(p)[i];
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[i * kPer + j] = K::to_f32(v.e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = K::to_f32(p[i]);
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

// One workgroup per touched block of a sequence and head. Keys are the first
// pass, values the second: the new rows' largest magnitude over the workgroup,
// the block's scale, then its bytes in page order. Values are transposed
// through LDS. Bound by the bytes of the rows and codes.
template <int TYPE, int D>
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(AppendArgs a) {
    using T = typename KvType<TYPE>::T;
    constexpr int kChunks = kKvBlock * D / 16;                               // 16-byte pieces of keys, and of values
    constexpr int kRounds = (kChunks + kAppendThreads - 1) / kAppendThreads;
    __shared__ uint32_t red[2][kAppendThreads / 64];
    __shared__ alignas(16) int8_t codes[kKvBlock][D + 4];
    const int tid = threadIdx.x, b = blockIdx.z, h = blockIdx.y;
    const KvSpan s = kv_span(a.past, a.cu, b, a.rows, a.max_new);
    const int j = s.past / kKvBlock + blockIdx.x;
    const int lead = max(s.past - j * kKvBlock, 0);          // tokens the block held before
    const int end = min(s.past + s.n - j * kKvBlock, kKvBlock);
    if (end <= lead) return;
    const int64_t entry_row = (static_cast<int64_t>(b) * a.c.kv_heads + h) * a.c.max_blocks;
    const int at = j - a.c.dropped[b];
    if (at < 0 || at >= a.c.max_blocks) return;
    const int page = a.c.table[entry_row + at];
    if (page < 0 || page >= a.c.n_pages) return;
    uint8_t* keys = a.c.pages + static_cast<int64_t>(page) * (2 * kKvBlock * D);
    const int64_t row = s.row0 + (j * kKvBlock - s.past);     // the row of the block's token 0

    float x[2][kRounds][16];
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const T* src = static_cast<const T*>(w ? a.v : a.k) + h * (w ? a.v_head : a.k_head);
        const int64_t stride = w ? a.v_row : a.k_row;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = tid + r * kAppendThreads, t = i / (D / 16), c = i % (D / 16);
            if (t >= lead && t < end) {
                load16<TYPE>(src + (row + t) * stride + c * 16, a.vec, x[w][r]);
#pragma unroll
                for (int e = 0; e < 16; ++e) top[w] = max(top[w], __float_as_uint(x[w][r][e]) & 0x7fffffffu);
            }
        }
        top[w] = wave_max_u32(top[w]);
        if ((tid & 63) == 0) red[w][tid >> 6] = top[w];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        top[w] = red[w][0];
#pragma unroll
        for (int i = 1; i < kAppendThreads / 64; ++i) top[w] = max(top[w], red[w][i]);
        const float before = lead > 0 ? a.c.scales[2 * static_cast<int64_t>(page) + w] : 0.0f;
        const float amax = __uint_as_float(top[w]);
        // bit patterns above FLT_MAX are infinities and NaNs
        const bool bad = top[w] > 0x7f7fffffu || !(before <= 3.402823466e38f);
        const float scale = bad ? __builtin_nanf("") : fmaxf(fmaxf(amax / 127.0f, before), kKvScaleFloor);
        const float inv = bad ? 0.0f : 1.0f / scale, again = bad ? 0.0f : before / scale;
        int8_t* out = reinterpret_cast<int8_t*>(keys) + w * (kKvBlock * D);
        // new codes: keys straight to their place, values to LDS
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = tid + r * kAppendThreads, t = i / (D / 16), c = i % (D / 16);
            if (t >= lead && t < end) {
                alignas(16) int8_t q[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) q[e] = bad ? int8_t{0} : code_of(x[w][r][e], inv);
                if (w == 0) {
                    *reinterpret_cast<uint4*>(out + kv_key_at(t, c * 16)) = *reinterpret_cast<uint4*>(q);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        reinterpret_cast<uint32_t*>(&codes[t][c * 16])[e] = reinterpret_cast<uint32_t*>(q)[e];
                }
            } else if (w == 0 && t < lead && again != 1.0f) {
                alignas(16) int8_t q[16];
                *reinterpret_cast<uint4*>(q) = *reinterpret_cast<uint4*>(out + kv_key_at(t, c * 16));
#pragma unroll
                for (int e = 0; e < 16; ++e) q[e] = code_of(static_cast<float>(q[e]), again);
                *reinterpret_cast<uint4*>(out + kv_key_at(t, c * 16)) = *reinterpret_cast<uint4*>(q);
            }
        }
        if (w == 1) {
            __syncthreads();
            // values in page order: 16 bytes are 8 tokens of dims d and d + 16
            for (int i = tid; i < kChunks; i += kAppendThreads) {
                const int d = i / 64 * 32 + i / 4 % 16, t4 = i % 4 * 4;
                alignas(16) int8_t q[16];
                if (lead > 0) *reinterpret_cast<uint4*>(q) = *reinterpret_cast<uint4*>(out + i * 16);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int t = e / 4 % 2 * 16 + t4 + e % 4;
                    if (t < lead)
                        q[e] = code_of(static_cast<float>(q[e]), again);
                    else
                        q[e] = t < end ? codes[t][d + e / 8 * 16] : int8_t{0};
                }
                *reinterpret_cast<uint4*>(out + i * 16) = *reinterpret_cast<uint4*>(q);
            }
        }
        // all threads have read the scale before it is replaced
        __syncthreads();
        if (tid == 0) a.c.scales[2 * static_cast<int64_t>(page) + w] = scale;
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

// One workgroup per 32 positions of a sequence and head, a thread per 16 dims
// of a position.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(rocknpu_kv_cache c, const int32_t* __restrict__ first,
                                                      const int32_t* __restrict__ tokens, int64_t count,
                                                      typename KvType<TYPE>::T* __restrict__ k,
                                                      typename KvType<TYPE>::T* __restrict__ v) {
    using K = KvType<TYPE>;
    using T = typename K::T;
    const int b = blockIdx.z, h = blockIdx.y;
    const int total = min(max(tokens[b], 0), 0x3fffffff);
    const int gone = max(c.dropped[b], 0);
    const int held = min((total + kKvBlock - 1) / kKvBlock - gone, c.max_blocks);
    const int64_t entry_row = (static_cast<int64_t>(b) * c.kv_heads + h) * c.max_blocks;
    for (int i = threadIdx.x; i < kKvBlock * D / 16; i += 256) {
        const int64_t o = static_cast<int64_t>(blockIdx.x) * kKvBlock + i / (D / 16);
        const int d = i % (D / 16) * 16;
        if (o >= count) continue;
        const int64_t pos = first[b] + o;
        float xk[16] = {}, xv[16] = {};
        if (pos >= 0 && pos < total) {
            const int start = static_cast<int>(pos) / kKvBlock * kKvBlock, t = static_cast<int>(pos) % kKvBlock;
            int at = start / kKvBlock;
            if (gone) at = find_block(c.starts + entry_row, held, start);
            const int page = at >= 0 && at < held ? c.table[entry_row + at] : -1;
            if (page >= 0 && page < c.n_pages) {
                const int8_t* keys = reinterpret_cast<const int8_t*>(c.pages) + static_cast<int64_t>(page) * (2 * kKvBlock * D);
                const int8_t* values = keys + kKvBlock * D;
                const float sk = c.scales[2 * static_cast<int64_t>(page)], sv = c.scales[2 * static_cast<int64_t>(page) + 1];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    xk[e] = static_cast<float>(keys[kv_key_at(t, d + e)]) * sk;
                    xv[e] = static_cast<float>(values[kv_value_at(t, d + e)]) * sv;
                }
            }
        }
        const int64_t to = ((static_cast<int64_t>(b) * count + o) * c.kv_heads + h) * D + d;
        struct alignas(16) Quad {
            T e[16 / sizeof(T)];
        };
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int p = 0; p < 16 / kPer; ++p) {
            Quad qk, qv;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                qk.e[e] = K::from_f32(xk[p * kPer + e]);
                qv.e[e] = K::from_f32(xv[p * kPer + e]);
            }
            reinterpret_cast<Quad*>(k + to)[p] = qk;
            reinterpret_cast<Quad*>(v + to)[p] = qv;
        }
    }
}

// An order-preserving map of weights to whole numbers: NaN is 0, -0 equals +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of `v` over the threads before this one; `total` over all of them.
template <int THREADS>
__device__ __forceinline__ int exclusive_sum(int v, int* part, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    __syncthreads();
    return before + x - v;
}

// One workgroup per row of the table, every thread with ITEMS consecutive
// entries in registers. The budget-th greatest key is found a byte at a time
// from the top (a histogram of the entries that match the bytes found so far),
// then two sums over the threads place every entry. Everything is read before
// the first write, so outputs may be the inputs. Bound by the latency of its
// steps: a row is a few kilobytes.
template <int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void kv_evict_kernel(rocknpu_kv_evict_args a) {
    __shared__ int hist[256];
    __shared__ int part[THREADS / 64];
    __shared__ int pick[2];  // the byte found, and how many entries rank above it
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int b = static_cast<int>(r / a.kv_heads);
    const int64_t base = r * a.max_blocks;
    const int total = min(max(a.tokens[b], 0), 0x3fffffff);
    const int gone = max(a.dropped[b], 0);
    const int n = min(max((total + kKvBlock - 1) / kKvBlock - gone, 0), a.max_blocks);
    int32_t page[ITEMS], start[ITEMS];
    float w[ITEMS];
    uint32_t key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int at = tid * ITEMS + i;
        const bool in = at < a.max_blocks;
        page[i] = in ? a.table[base + at] : 0;
        start[i] = in ? a.starts[base + at] : 0;
        w[i] = in ? a.weights[base + at] : 0.0f;
        key[i] = at < a.sinks || at >= n - a.recent ? 0xffffffffu : weight_key(w[i]);
    }
    __syncthreads();
    if (n > a.budget) {
        uint32_t found = 0;
        int above = 0;  // entries known to rank above the budget-th
#pragma unroll
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (tid * ITEMS + i < n && (shift == 24 || key[i] >> ((shift + 8) & 31) == found))
                    atomicAdd(&hist[key[i] >> shift & 255], 1);
            __syncthreads();
            if (tid < 64) {  // lane l: bins 255 - 4 l down to 252 - 4 l
                int c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += c[i] = hist[255 - 4 * tid - i];
                int x = sum;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int y = __shfl_up(x, o, 64);
                    if (tid >= o) x += y;
                }
                int up = above + x - sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (up < a.budget && up + c[i] >= a.budget) {
                        pick[0] = 255 - 4 * tid - i;
                        pick[1] = up;
                    }
                    up += c[i];
                }
            }
            __syncthreads();
            found = found << 8 | static_cast<uint32_t>(pick[0]);
            above = pick[1];
        }
        // of the entries equal to the budget-th key the first budget - above stay
        int equal = 0, kept = 0, sum;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) equal += tid * ITEMS + i < n && key[i] == found;
        int rank = exclusive_sum<THREADS>(equal, part, sum);
        bool keep[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool in = tid * ITEMS + i < n;
            keep[i] = in && (key[i] > found || (key[i] == found && rank < a.budget - above));
            rank += in && key[i] == found;
            kept += keep[i];
        }
        int before = exclusive_sum<THREADS>(kept, part, sum);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = tid * ITEMS + i;
            const int to = at >= n ? at : keep[i] ? before : a.budget + at - before;
            before += keep[i];
            if (at < a.max_blocks) {
                a.table_out[base + to] = page[i];
                a.starts_out[base + to] = start[i];
                a.weights_out[base + to] = w[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = tid * ITEMS + i;
            if (at < a.max_blocks) {
                a.table_out[base + at] = page[i];
                a.starts_out[base + at] = start[i];
                a.weights_out[base + at] = w[i];
            }
        }
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
    const dim3 grid(static_cast<unsigned>((count + kKvBlock - 1) / kKvBlock), c.kv_heads, c.batch);
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
