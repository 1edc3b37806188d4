// What the kernels of the 8-bit key/value cache share: a block's byte layout,
// a step's lengths as the device reads them, and element conversions.
//
// A page (include/rocknpu_kv.h) holds 32 tokens of one kv head, keys then
// values. The orders are those in which a wave's lanes feed the matrix
// instructions: for v_mfma_f32_16x16x32_f16 lane l = 16 q + r supplies 8
// contraction values of row r. Keys are the first operand of the scores
// (row = token, contraction = dims): lane (r, q) loads the 16 bytes of dims
// 64 c + 16 q .. + 15 of token r, two instructions' worth. Values are the first
// operand of the output (row = dim, contraction = tokens): the scores leave
// their instruction with lane (., q) holding tokens 4 q + 0..3 of each 16-token
// tile, so a lane's 8 contraction values are those tokens of both tiles, and 16
// bytes serve dims d and d + 16.
#pragma once

#include "common.h"
#include "rocknpu_kv.h"

namespace rk {

constexpr int kKvBlock = 32;
constexpr float kKvScaleFloor = 0x1p-100f;
constexpr int kKvMaxWeightRows = 256;
constexpr int kKvMaxBatch = 4095;  // sequences, or their slots (a few thousand more), are a grid's z, which ends at 65535
constexpr int kKvEvictMaxBlocks = 16384;

template <int TYPE>
struct KvType;
template <>
struct KvType<ROCKNPU_KV_F32> {
    using T = float;
    static __device__ __forceinline__ float to_f32(T x) { return x; }
    static __device__ __forceinline__ T from_f32(float x) { return x; }
};
template <>
struct KvType<ROCKNPU_KV_F16> {
    using T = _Float16;
    static __device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }
    static __device__ __forceinline__ T from_f32(float x) { return static_cast<T>(x); }
};
template <>
struct KvType<ROCKNPU_KV_BF16> {
    using T = __bf16;
    static __device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }
    static __device__ __forceinline__ T from_f32(float x) { return static_cast<T>(x); }
};

// A sequence's part of a step: `past` tokens before it, rows row0 .. row0 + n - 1.
// Whatever past and cu hold, the rows lie inside the step's tensors.
struct KvSpan {
    int past, row0, n;
};
// The four are asked for before any is waited for, and before a branch on one of
// them: a kernel's start is a chain of trips to memory, this makes them one.
__device__ __forceinline__ KvSpan kv_span(const int32_t* past, const int32_t* cu, const int32_t* dropped, int b, int rows,
                                          int max_new, int& gone) {
    int had = past[b], first = cu[b], last = cu[b + 1], lost = dropped[b];
    asm volatile("" : "+v"(had), "+v"(first), "+v"(last), "+v"(lost));
    KvSpan s;
    s.past = min(max(had, 0), 0x3fffffff);
    s.row0 = min(max(first, 0), rows);
    const int end = min(max(last, s.row0), rows);
    s.n = min(end - s.row0, max_new);
    gone = max(lost, 0);
    return s;
}

// A value that is the same in every lane, into a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ KvSpan uniform(KvSpan s) { return KvSpan{uniform(s.past), uniform(s.row0), uniform(s.n)}; }

// Lane l gets the sum over lanes 0 .. l: four steps within rows of 16 lanes, then
// lane 15 of the odd rows' predecessors and lane 31 into what follows them.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 to rows 2 and 3
    return x;
}

// Whether a cache description is one that the kernels can take. kv_cache.hip.
bool kv_cache_ok(const rocknpu_kv_cache* c);

}  // namespace rk
