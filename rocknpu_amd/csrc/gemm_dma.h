// What the kernels that feed int8 MFMA tiles by direct global->LDS loads share:
// the stage layout, the loads and the waits.
#pragma once

#include "common.h"

#include <type_traits>
#include <utility>

namespace rk {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// Direct-load tiles: the same product with a pipeline of ST (2 to 8) LDS
// stage buffers filled by direct global->LDS loads (global_load_lds_dwordx4,
// no register staging). A stage holds KB (64 or 128) bytes of K per row. Each
// wave issues its share of a stage as 1 KiB segments (1024 / KB rows of KB
// bytes; lane i's 16 bytes land at segment + 16*i, so the lane loads the
// global chunk that the swizzled layout puts there). Stage s+ST-1 is issued
// while stage s is multiplied; one barrier per stage both publishes stage s+1
// (after each wave's own wait for its loads) and frees stage s for reuse. The
// barrier is a bare s_barrier: a fenced one would wait for every load in
// flight, stages ahead included.
template <int BM, int BN, int WM, int WN, int KB>
struct DmaTile {
    static constexpr int T = WM * WN * 64;
    static constexpr int W = WM * WN;
    // 1 KiB segments (RPI rows of KB bytes) per wave and stage. When a tile
    // has fewer segments than waves, waves load segments twice (the same
    // bytes to the same LDS place), so every wave issues the same number of
    // loads.
    static constexpr int RPI = 1024 / KB;
    static constexpr int A_ROWSEG = BM / RPI, B_ROWSEG = BN / RPI;
    static constexpr int A_SEG = A_ROWSEG >= W ? A_ROWSEG / W : 1, B_SEG = B_ROWSEG >= W ? B_ROWSEG / W : 1;
    static_assert(BM % RPI == 0 && BN % RPI == 0, "tile rows must split into whole segments");
    static_assert((B_ROWSEG >= W ? B_SEG * W == B_ROWSEG : W % B_ROWSEG == 0) &&
                      (A_ROWSEG >= W ? A_SEG * W == A_ROWSEG : W % A_ROWSEG == 0),
                  "segments split evenly over the waves");
};

// s_waitcnt with only vmcnt constrained (gfx9 encoding: vmcnt[3:0] | expcnt[6:4]
// | lgkmcnt[11:8] | vmcnt[5:4] at bits 15:14).
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xF | (7 << 4) | ((0x3) << 14)); }

// Stage layout of the direct-load tiles: rows of KB bytes (64 or 128), the
// 16-byte chunks XOR-swizzled by row / 2, so the fragment reads (32 rows,
// one chunk column per half wave) do not collide in the LDS banks.
template <int KB>
__device__ __forceinline__ int swz_kb(int r, int kc) { return r * KB + ((kc ^ ((r >> 1) & (KB / 16 - 1))) << 4); }

// One 16-byte direct global->LDS load per lane; `lds` must be wave-uniform
// (the 64 lanes fill lds .. lds + 1023).
__device__ __forceinline__ void dma16(const int8_t* src, int8_t* lds) {
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)(lds), 16, 0, 0);
}

// Calls f(integral_constant<int, I>) for I in the sequence, in order.
template <typename F, int... I>
__device__ __forceinline__ void unroll_seq(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

}  // namespace rk
