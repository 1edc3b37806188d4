// The experts' W8A8 products: grouped by the routing's plan, gate and up in one
// pass with SwiGLU.
//
// out[r][c] = (f32(sum_k A[row of r][k] * W[e][c][k]) * a_scale) * w_scale for
// every row r in order of expert (e is its expert), or for gate and up together
// out[r][c] = f32(g * u / (1 + exp(-g))). Sums are exact int32.
//
// Tiling, stages and waits are gemm.hip's: BM x BN tiles of 32x32 fragments of
// v_mfma_i32_32x32x32_i8, operands through LDS stage buffers that direct loads
// fill. What differs:
//   - A workgroup takes a tile of the plan: up to BM rows of one expert. For gate
//     and up the rows are gathered: each lane's source addresses are looked up
//     once, the direct loads take any.
//   - An expert's last tile has fewer rows. Rows are dealt to the WM waves of a
//     column by fragments of 32 in turn, so a tile of at most BM' rows runs as a
//     BM' x BN tile on the same buffers: fewer loads, reads and products.
//   - Gate's and up's columns alternate by fragments of 32 in a tile, so a lane
//     holds g and u of the same output, and no pass over [rows][2 ffn] follows.
//
// Measured, us (gate and up; down): 4096 tokens, top 8 of 64 experts of 2048 x 1024,
// 32768 rows: 235; 142. 2048 tokens, top 2 of 8 of 4096 x 14336: 620; 310, 1.5 POP/s
// (gemm.hip on one matrix of gate's and up's size: 462 to 525, by 16 full row tiles; here
// 16 to 24 are begun, 19 in that call, and SwiGLU and a tile's start are 15 us of a
// tile's 71). 64 tokens of the latter: 187; 82, 5.0 and 5.7 TB/s of weights.
//   - 256 x 256 tiles by eight waves of 128 x 64, two a SIMD; by four waves of 128 x 128
//     252; 160 and 630; 319. 256 x 128 tiles, two workgroups a CU, whose epilogues overlap
//     with each other's products: 250; 165 and 671; 376.
//   - 64 x 128 tiles by two waves, three stages, two workgroups a CU; 64 x 64 tiles by one
//     wave 184; 85 (333 tokens of 24 experts 33; 20 against 26; 16), two stages 188; 110, 64 x
//     256 tiles by four waves 181; 103.
//   - What bounds a 256 x 256 gate tile of K = 2048 (46 us): its products at the rate of a
//     long product (28), SwiGLU's 64-bit operations (10), and its start, a chain of
//     lookups and the first stage (5); of a down tile of K = 1024 (28 us) the products are
//     14, the rest is mostly the 256 KiB that every CU writes at the same time.
#include "gemm_dma.h"
#include "moe.h"
#include "moe_product.h"

namespace rk {
namespace {

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// One tile: rows r0 .. end - 1 (at most BME) of the plan's order, expert e, output
// columns from c0. `stages(A?, stage)` names the stage buffers, distinct arrays, so
// that a wait for one does not wait for all.
template <int BME, int BN, int WM, int WN, int ST, int KB, bool GATED, typename SA, typename SB>
__device__ __forceinline__ void product_tile(const MoeProduct& p, const int32_t* __restrict__ order, int rows, int e, int r0,
                                             int end, int c0, SA stage_a, SB stage_b, float* lsc) {
    using Cfg = DmaTile<BME, BN, WM, WN, KB>;
    constexpr int TN = BN / WN, FM = BME / WM / 32, FN = TN / 32;
    constexpr int CPR = KB / 16, THREADS = WM * WN * 64;
    static_assert(FM * WM * 32 == BME && FN * WN * 32 == BN && (!GATED || FN % 2 == 0), "whole fragments, gate's and up's in pairs");
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int k = p.k;
    // the row of A behind tile row r: rows past the tile re-read its last one
    const auto source = [&](int r) {
        const int at = min(r0 + r, end - 1);
        return GATED ? min(max(order[at], 0), rows - 1) / p.top_k : at;
    };
    // the row of W (of which matrix) behind tile column c; columns past the matrix re-read its last one
    const auto column = [&](int c) { return min(c0 + (GATED ? (c >> 6) * 32 + (c & 31) : c), p.n - 1); };
    const int64_t first = static_cast<int64_t>(e) * p.n;

    // Addresses of the direct loads: a base that is the same for the wave and 32 bits
    // a lane (half the registers and none of the additions of 64-bit pointers). A
    // segment's rows lie in one fragment, so in one matrix.
    const int8_t* abase = GATED ? p.a : p.a + static_cast<int64_t>(r0) * k;
    const int8_t* bbase[Cfg::B_SEG];
    uint32_t aoff[Cfg::A_SEG], boff[Cfg::B_SEG];
#pragma unroll
    for (int q = 0; q < Cfg::A_SEG; ++q) {
        const int r = ((wave * Cfg::A_SEG + q) % Cfg::A_ROWSEG) * Cfg::RPI + lane / CPR;
        const int c = (lane % CPR) ^ ((r >> 1) & (CPR - 1));
        aoff[q] = static_cast<uint32_t>(source(r) - (GATED ? 0 : r0)) * static_cast<uint32_t>(k) + c * 16;
    }
#pragma unroll
    for (int q = 0; q < Cfg::B_SEG; ++q) {
        const int r0q = ((wave * Cfg::B_SEG + q) % Cfg::B_ROWSEG) * Cfg::RPI, r = r0q + lane / CPR;
        const int c = (lane % CPR) ^ ((r >> 1) & (CPR - 1));
        bbase[q] = (GATED && (r0q & 32) ? p.w[1] : p.w[0]) + (first + c0) * k;
        boff[q] = static_cast<uint32_t>(column(r) - c0) * static_cast<uint32_t>(k) + c * 16;
    }
    auto issue = [&](auto st, int ks) {
        int8_t* la = stage_a(st);
        int8_t* lb = stage_b(st);
        const int at = ks * KB;
#pragma unroll
        for (int q = 0; q < Cfg::A_SEG; ++q)
            dma16(abase + at + aoff[q], la + ((wave * Cfg::A_SEG + q) % Cfg::A_ROWSEG) * 1024);
#pragma unroll
        for (int q = 0; q < Cfg::B_SEG; ++q)
            dma16(bbase[q] + at + boff[q], lb + ((wave * Cfg::B_SEG + q) % Cfg::B_ROWSEG) * 1024);
    };

    v16i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v16i{};

    // A step multiplies 64 bytes of K, two 32-deep halves, while the fragments of the next
    // step are read into the other register set.
    constexpr int D = 2;
    constexpr int SUB = KB / (32 * D);  // steps of a stage
    const int KS = k / KB;              // stages
    const int KT = KS * SUB;            // steps
    using S0 = std::integral_constant<int, 0>;
    using R0 = std::integral_constant<int, 0>;
    constexpr int PER_STAGE = Cfg::A_SEG + Cfg::B_SEG;
    v4i fa[2][D][FM], fb[2][D][FN];  // [register set][32-deep half][fragment]
    // lane l supplies row l % 32 and the 16 bytes of chunk 2 h + l / 32 of half h; fragment i
    // of wave column wm holds tile rows 32 (WM i + wm) .. A row's swizzle is the same in every
    // fragment, and another half's place is an exclusive or away: worked out where it is
    // read (an asm, or the compiler would keep all of them in registers that the
    // accumulators leave no room for).
    const int a0 = swz_kb<KB>(wm * 32 + (lane & 31), half), b0 = swz_kb<KB>(wn * TN + (lane & 31), half);
    const auto at_half = [](int base, auto h) {
        int at;
        asm volatile("v_xor_b32 %0, %1, %2" : "=v"(at) : "i"(decltype(h)::value * 32), "v"(base));
        return at;
    };
    auto read_frags = [&](auto st, auto set, auto u) {
        constexpr int R = decltype(set)::value, SU = decltype(u)::value;
        const int8_t* la = stage_a(st);
        const int8_t* lb = stage_b(st);
        unroll_seq([&](auto h) {
            constexpr int H = decltype(h)::value;
            using Half = std::integral_constant<int, D * SU + H>;
            const int pa = at_half(a0, Half{}), pb = at_half(b0, Half{});
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[R][H][i] = *reinterpret_cast<const v4i*>(la + pa + i * WM * 32 * KB);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[R][H][j] = *reinterpret_cast<const v4i*>(lb + pb + j * 32 * KB);
        }, std::make_integer_sequence<int, D>{});
    };
    auto mfma = [&](auto set) {
        constexpr int R = decltype(set)::value;
#pragma unroll
        for (int h = 0; h < D; ++h)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[R][h][i], fb[R][h][j], acc[i][j], 0, 0, 0);
    };
    // The tile's scales: each thread loads one or two before the stages (older than
    // their loads, so the waits' counts hold) and writes them to LDS once the first
    // stage has landed; the loop's barriers publish them.
    constexpr int NSC = BME + BN, SCP = (NSC + THREADS - 1) / THREADS;
    float scv[SCP];
#pragma unroll
    for (int u = 0; u < SCP; ++u) {
        const int idx = threadIdx.x + u * THREADS, c = min(idx, NSC - 1) - BME;
        const float* sc = idx < BME ? p.a_scales + source(idx) : (GATED && (c & 32) ? p.w_scales[1] : p.w_scales[0]) + first + column(c);
        scv[u] = *sc;
    }
    // prologue: stages 0 .. ST-2 in flight, wait for stage 0, then stage ST-1
    unroll_seq([&](auto i) { issue(i, min(static_cast<int>(decltype(i)::value), KS - 1)); }, std::make_integer_sequence<int, ST - 1>{});
    wait_vm<(ST - 2) * PER_STAGE>();
#pragma unroll
    for (int u = 0; u < SCP; ++u) {
        const int idx = threadIdx.x + u * THREADS;
        if (idx < NSC) lsc[idx] = scv[u];
    }
    __builtin_amdgcn_s_barrier();
    issue(std::integral_constant<int, ST - 1>{}, min(ST - 1, KS - 1));
    read_frags(S0{}, R0{}, S0{});
    // A step, as in gemm.hip: the fragments of step j were read in step j-1;
    // the last step of a stage waits for the next one, passes the barrier that frees
    // the stage's buffer, and refills it.
    auto step = [&](auto set, auto next_st, auto next_u, auto refill_st, auto last_of_stage, int q) {
        using NSET = std::integral_constant<int, 1 - decltype(set)::value>;
        constexpr bool LAST = decltype(last_of_stage)::value;
        wait_lgkm0();
        if constexpr (LAST) {
            wait_vm<(ST - 2) * PER_STAGE>();
            __builtin_amdgcn_s_barrier();
            issue(refill_st, min(q + ST, KS - 1));
        }
        read_frags(next_st, NSET{}, next_u);
        mfma(set);
        constexpr int READS = D * (FM + FN), MFMAS = D * FM * FN;
        if constexpr (LAST && READS % PER_STAGE == 0 && MFMAS % PER_STAGE == 0) {
#pragma unroll
            for (int i = 0; i < PER_STAGE; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);                  // VMEM read (direct load)
                __builtin_amdgcn_sched_group_barrier(0x100, READS / PER_STAGE, 0);  // DS read
                __builtin_amdgcn_sched_group_barrier(0x008, MFMAS / PER_STAGE, 0);  // MFMA
            }
        } else if constexpr (!LAST && MFMAS % READS == 0) {
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);              // DS read
                __builtin_amdgcn_sched_group_barrier(0x008, MFMAS / READS, 0);  // MFMA
            }
        }
    };
    auto step_i = [&](auto i, int kt) {
        constexpr int I = decltype(i)::value;
        step(std::integral_constant<int, I % 2>{}, std::integral_constant<int, ((I + 1) / SUB) % ST>{},
             std::integral_constant<int, (I + 1) % SUB>{}, std::integral_constant<int, (I / SUB) % ST>{},
             std::integral_constant<bool, (I + 1) % SUB == 0>{}, (kt + I) / SUB);
    };
    constexpr int U = (ST * SUB) % 2 == 0 ? ST * SUB : 2 * ST * SUB;
    const int KTA = KT - KT % U;
    for (int kt = 0; kt < KTA; kt += U) unroll_seq([&](auto i) { step_i(i, kt); }, std::make_integer_sequence<int, U>{});
    unroll_seq([&](auto i) { if (KTA + decltype(i)::value < KT) step_i(i, KTA); }, std::make_integer_sequence<int, U - 1>{});
    wait_vm<0>();  // no direct load is in flight when the workgroup's LDS is given back
    wait_lgkm0();

    // Epilogue. lane l holds column l % 32 of each fragment, rows (i % 4) + 4 (l / 32) +
    // 8 (i / 4): a store is two whole runs of 128 bytes. Eight values at a time, so that
    // their chains of 64-bit operations overlap.
    constexpr int STEP = GATED ? 2 : 1, X = 8;
    float* out = p.out + static_cast<int64_t>(r0) * p.ldo + c0;
#pragma unroll
    for (int j = 0; j < FN; j += STEP) {
        const int tc = wn * TN + j * 32 + (lane & 31);
        const int col = GATED ? (tc >> 6) * 32 + (tc & 31) : tc;
        const float ws0 = lsc[BME + tc], ws1 = GATED ? lsc[BME + tc + 32] : 0.0f;
        const int last = c0 + col < p.ldo ? end - r0 : 0;
        const bool inside = c0 + col < p.n;  // zeros behind it, up to the rows' length
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int x0 = 0; x0 < 16; x0 += X) {
                float v[X];
#pragma unroll
                for (int x = 0; x < X; ++x) {
                    const int f = x0 + x;
                    const float as = lsc[(i * WM + wm) * 32 + (f & 3) + 4 * half + 8 * (f >> 2)];
                    v[x] = (static_cast<float>(acc[i][j][f]) * as) * ws0;
                    if constexpr (GATED) v[x] = swiglu(v[x], (static_cast<float>(acc[i][j + STEP - 1][f]) * as) * ws1);
                }
                // all of them before the first store's condition, or each would wait for its own chain
                asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]));
#pragma unroll
                for (int x = 0; x < X; ++x) {
                    const int f = x0 + x, r = (i * WM + wm) * 32 + (f & 3) + 4 * half + 8 * (f >> 2);
                    if (r < last) out[static_cast<uint32_t>(r * p.ldo + col)] = inside ? v[x] : 0.0f;
                }
            }
        }
    }
}

template <int BM, int BN, int WM, int WN, int ST, int KB, bool GATED>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(const MoeProduct p, const MoePlan plan) {
    static_assert(ST >= 2 && ST <= 4, "two to four stage buffers");
    __shared__ __align__(16) int8_t la0[BM * KB], la1[BM * KB], la2[ST > 2 ? BM * KB : 16], la3[ST > 3 ? BM * KB : 16];
    __shared__ __align__(16) int8_t lb0[BN * KB], lb1[BN * KB], lb2[ST > 2 ? BN * KB : 16], lb3[ST > 3 ? BN * KB : 16];
    __shared__ float lsc[BM + BN];
    auto stage_a = [&](auto st) -> int8_t* {
        constexpr int S = decltype(st)::value;
        if constexpr (S == 0) return la0; else if constexpr (S == 1) return la1;
        else if constexpr (S == 2) return la2; else return la3;
    };
    auto stage_b = [&](auto st) -> int8_t* {
        constexpr int S = decltype(st)::value;
        if constexpr (S == 0) return lb0; else if constexpr (S == 1) return lb1;
        else if constexpr (S == 2) return lb2; else return lb3;
    };
    constexpr int BC = GATED ? BN / 2 : BN;  // output columns of a tile
    const int tiles_m = uniform(max(min(*plan.tile_count, plan.max_tiles), 0));
    const MoeShare share = moe_share(blockIdx.x & 7, tiles_m, (p.n + BC - 1) / BC, p.xcd_cus, BM == 256);
    int i = blockIdx.x >> 3, part, tm, tn;
    moe_part(share, i, part);
    if (i >= share.mine) return;
    moe_pair(share, i, tm, tn);
    const int e = uniform(min(max(plan.tiles[2 * tm], 0), plan.experts - 1));
    int r0 = uniform(min(max(plan.tiles[2 * tm + 1], 0), plan.rows));
    int end = uniform(min(min(plan.offsets[e + 1], plan.rows), r0 + BM));
    const int c0 = tn * BC;
    if constexpr (BM == 256)
        // (not that it is likely: the compiler then puts the parts' code before the whole
        // tiles', 425 us against 429 for 4096 tokens of 64 small experts)
        if (__builtin_expect(moe_splits(share, i), true)) {
            r0 += part / 2 * (BM / 2);
            if (share.parts == 4) end = min(end, r0 + BM / 2);
            const int c1 = c0 + part % 2 * (BC / 2), n = end - r0;
            if (n <= 0 || c1 >= p.n) return;
#define RK_PART(BME) product_tile<BME, BN / 2, WN, WM, ST, KB, GATED>(p, plan.order, plan.rows, e, r0, end, c1, stage_a, stage_b, lsc)
            if (n > 128) return RK_PART(256);
            return RK_PART(128);
#undef RK_PART
        }
    const int n = end - r0;
    if (n <= 0) return;
#define RK_TILE(BME) product_tile<BME, BN, WM, WN, ST, KB, GATED>(p, plan.order, plan.rows, e, r0, end, c0, stage_a, stage_b, lsc)
    if constexpr (BM == 256) {
        // (192 rows of 64 bytes are not whole segments for 8 waves)
        if (n > (KB == 128 ? 192 : 128)) return RK_TILE(256);
        if constexpr (KB == 128)
            if (n > 128) return RK_TILE(192);
        if (n > 64) return RK_TILE(128);
        return RK_TILE(64);
    } else {
        if (n > 32) return RK_TILE(64);
        return RK_TILE(32);
    }
#undef RK_TILE
}

template <int BM, int BN, int WM, int WN, int ST, int KB, bool GATED>
int launch(const MoeProduct& p, const MoePlan& plan, hipStream_t stream) {
    static_assert(moe_tile_columns(BM, GATED) == (GATED ? BN / 2 : BN), "the grid is worked out for these tiles");
    const int64_t grid = moe_product_grid(plan, p.n, GATED, p.xcd_cus);
    if (grid * (WM * WN * 64) > 0xffffffff) return kStatusInvalid;  // (values of that many tiles are over a TB)
    product_kernel<BM, BN, WM, WN, ST, KB, GATED><<<dim3(static_cast<unsigned>(grid)), dim3(WM * WN * 64), 0, stream>>>(p, plan);
    return hipGetLastError() == hipSuccess ? kStatusOk : kStatusExec;
}

template <bool GATED>
int route(const MoeProduct& p, const MoePlan& plan, hipStream_t stream) {
    // 128-byte stages need K % 128 == 0 (a stage never reads past a row)
    if (plan.tile_rows == 256) {
        if (p.k % 128 == 0) return launch<256, 256, 2, 4, 2, 128, GATED>(p, plan, stream);
        return launch<256, 256, 2, 4, 4, 64, GATED>(p, plan, stream);
    }
    if (p.k % 128 == 0) return launch<64, 128, 1, 2, 3, 128, GATED>(p, plan, stream);
    return launch<64, 128, 1, 2, 4, 64, GATED>(p, plan, stream);
}

}  // namespace

int launch_moe_product(MoeProduct p, bool gated, const MoePlan& plan, hipStream_t stream) {
    p.xcd_cus = moe_xcd_cus(device_cu_count());
    return gated ? route<true>(p, plan, stream) : route<false>(p, plan, stream);
}

}  // namespace rk
