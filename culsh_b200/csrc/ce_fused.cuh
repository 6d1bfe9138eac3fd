// Gradient of the cross entropy for rows of up to 256 values of 16 bits: G does not leave the SM.
//
// A CTA keeps 128 entries of one side ("own": rows for dX, queries for dQ) and goes through the other, a tile at a time:  S = own . other^T into tensor memory,  G = 2^(c S + term)
// by the epilogue's threads and back into tensor memory as 16 bits,  O += G . other with G as the operand that lies in tensor memory.  The other side's tile is loaded once for
// both products: K along its rows for the first, across them for the second.  S is made again for the other gradient: 8 m n d operations in place of 6, against 6 bytes of G written and read
// for each of the m n entries.
//
// The factor of a query's entries is multiplied in where queries are the columns, and goes to the sums where they are the lanes.  It holds what the term, lse in powers of two as one float, leaves
// behind its last bit (as a part of the term, log2 of its magnitude, it would lose that again: all p of a query off by lse 2^-24, 5e-3 where lse is 1e5).  What is added to a score comes in the order of
// the losses' pass, the bias first: their difference from lse is then that of the same numbers.
// One warp loads, one issues the first products and one the second (a single one, issuing 16 MMAs a tile and waiting three times, held them up: 4,096 x 1M x 128 4.12 ms in place of 3.7), two groups of
// eight warps take the tiles in turn, a thread half the columns of a lane.  S and G have two places each: what an MMA writes over has been read by the epilogue long before, and the tensor pipe has
// another product to do while a G is made.  (G on top of S, in three places, 4.34 ms: the first product had to wait until the second one in front of it was done.)  dQ of that case takes 1.4 ms, bound
// by the reads of shared memory, which the first product takes alone (tensor pipe 69 %); dX 2.2, with the terms, factors and targets of the columns read beside (46 %).  Sums of more than 32,768 entries are split (the accumulators cut off,
// see tc_gemm.cuh) over units, and ce_finish_kernel adds them up: those of as many queries or rows at a time as 256 MB hold of (32,769 x 100,000 x 128 2.7 ms; dX by pieces of rows, with G in memory, 8.8).
#pragma once

#include <type_traits>

#include "tc_gemm.cuh"

namespace culsh_b200 {

constexpr float CE_LOG2E = 1.4426950408889634f;
template <typename T>
__device__ __forceinline__ float ce_float(T v) { return (float)v; }
__device__ __forceinline__ float ce_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int CE_HALF_SHIFT = 14;  // p of half precision is held times 2^14, down to 2^-38

// What a power of two brings the largest factor to [2^14, 2^15].
__device__ __forceinline__ int ce_scale_exponent(const uint32_t* amax) {
    const uint32_t bits = amax ? __ldcg(amax) : 0u;
    return bits == 0u ? 0 : min(max(14 + 127 - (int)(bits >> 23), -100), 100);
}

// 1 / T back by it, no infinity: a sum of 0 stays 0.
__device__ __forceinline__ float ce_scale_back(float inv_t, int exponent) { return fminf(ldexpf(inv_t, -exponent), 0x1.fffffep127f); }

// 32 rows of 32 values, a row to a lane, turned: lane i gets column i, v[j] that of row j.
__device__ __forceinline__ void ce_turn(float (&v)[32], int lane) {
#pragma unroll
    for (int s = 16; s; s >>= 1)
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (!(j & s)) {
                const bool high = lane & s;
                const float got = __shfl_xor_sync(0xFFFFFFFFu, high ? v[j] : v[j | s], s);
                if (high) v[j] = got;
                else v[j | s] = got;
            }
}
// Adds the sums of a row's targets, d columns each, over the temperature: 32 columns from `col` on.
__device__ __forceinline__ void ce_add_own(float (&v)[32], const int* where, int64_t stride, int splits, const float* sums, int d, int col, float inv_t) {
    for (int s = 0; s < splits; ++s) {
        const int slot = __ldcg(where + s * stride);
        if (slot < 0) continue;
        const float* const extra = sums + (int64_t)slot * d + col;
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (col + j < d) v[j] = fmaf(__ldcg(extra + j), inv_t, v[j]);
    }
}

struct CeFusedArgs {
    int* d_error;
    unsigned units;
    uint32_t idesc_s, idesc_o;
    int own, other;           // entries of either side
    int own0;                 // rows: the first one's number
    int tiles_own, tiles_other, block;
    int d;
    float c;
    const float* bias;        // of the rows, in powers of two, or NULL; in lines of 128
    // of the queries, for dX in lines of 128 with -inf, 0 and -1 behind the last one
    const float* terms;       // -lse in powers of two, in half precision CE_HALF_SHIFT more
    const float* factors;
    const int* target_cols;
    const uint32_t* amax;
    float* parts;             // sums: [block][own entry][d]; of dX NULL where they are complete
    void* out;                // dX
    int64_t ld;
    const int* where;
    int64_t where_stride;
    int own_splits;
    const float* sums;
    float inv_t;
};

// KB: boxes of 64 values in a row.
template <int KB>
struct CeFusedCfg {
    static constexpr int NB = KB == 4 ? 64 : 128;             // entries of a tile of the other side
    static constexpr int O_COLS = KB * 64, BUFS = 2, GROUPS = 2, WARPS = 8;  // of a group
    static constexpr int CW = NB / 2;                         // columns of a warp
    static constexpr int OWN_BYTES = KB * TG_M * 128, OWNS = KB == 1 ? 2 : 1;
    static constexpr int STAGE_BYTES = KB * NB * 128, COLUMN_BYTES = NB * 4, STAGES = KB == 1 ? 8 : KB == 2 ? 5 : 4;
    static constexpr int THREADS = 128 + 32 * WARPS * GROUPS;  // warps for the loads, either product, and one that idles
    static constexpr int COLUMNS = 3;  // terms, factors and targets, or the bias, of a stage's entries, which lie behind the stages
    // 640 threads are launched with 96 registers each; four warps give up some, which the others take: 128 x 32 + 512 x 112 = 640 x 96
    static constexpr int REGS = 96, FEW_REGS = 32, MANY_REGS = 112;
    static_assert(128 * FEW_REGS + 32 * WARPS * GROUPS * MANY_REGS <= THREADS * REGS, "");
    static constexpr int SMEM = OWNS * OWN_BYTES + STAGES * (STAGE_BYTES + COLUMNS * COLUMN_BYTES) + 1024 /*barriers*/ + 1024 /*alignment slack*/;
    static_assert(O_COLS + BUFS * (NB + NB / 2) <= 512 && SMEM <= 227 * 1024 && STAGES > BUFS, "");
};

__device__ __forceinline__ void tc_mma_ts_warp(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xFFFFFFFF;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tg_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tg_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// CTAs that work on units next to one another begin at different tiles: those that ask for the same lines at the same time wait for the few slices of L2 that hold them.
struct CeFusedUnit {
    int own0, tile0, tiles, block, turn;
    __device__ __forceinline__ CeFusedUnit(const CeFusedArgs& a, unsigned u) {
        block = (int)(u / (unsigned)a.tiles_own);
        own0 = (int)(u - (unsigned)block * a.tiles_own) * TG_M;
        tile0 = block * a.block;
        tiles = min(a.block, a.tiles_other - tile0);
        turn = (int)((int64_t)tiles * (u & 31u) >> 5);
    }
    __device__ __forceinline__ int tile(int t) const {
        t += turn;
        return tile0 + (t >= tiles ? t - tiles : t);
    }
};

template <int KB, bool ROWS, bool BIAS, bool HALF>
__global__ void __launch_bounds__(CeFusedCfg<KB>::THREADS, 1)
ce_fused_kernel(const __grid_constant__ CUtensorMap tmOwn, const __grid_constant__ CUtensorMap tmOther, CeFusedArgs a, KernelBefore before) {
    behind_kernel_before(before);
    using Cfg = CeFusedCfg<KB>;
    using T = std::conditional_t<HALF, __half, __nv_bfloat16>;
    constexpr int NB = Cfg::NB, BUFS = Cfg::BUFS, GROUPS = Cfg::GROUPS, STAGES = Cfg::STAGES, OWNS = Cfg::OWNS;
    extern __shared__ unsigned char cf_smem_raw[];
    unsigned char* const base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(cf_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* const s_other = base + OWNS * Cfg::OWN_BYTES;
    unsigned char* const s_columns = s_other + STAGES * Cfg::STAGE_BYTES;
    uint64_t* const own_full = reinterpret_cast<uint64_t*>(s_columns + STAGES * Cfg::COLUMNS * Cfg::COLUMN_BYTES);
    uint64_t* const own_empty = own_full + OWNS;
    uint64_t* const full = own_empty + OWNS;
    uint64_t* const empty = full + STAGES;
    uint64_t* const s_full = empty + STAGES;   // S is there
    uint64_t* const s_empty = s_full + BUFS;   // and has been read
    uint64_t* const g_full = s_empty + BUFS;   // G is there
    uint64_t* const g_empty = g_full + BUFS;   // and its product done
    uint64_t* const o_full = g_empty + BUFS;
    uint64_t* const o_empty = o_full + 1;
    uint64_t* const drained = o_empty + 1;
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    uint32_t* const s_fills = s_tmem + 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < OWNS; ++i) mbar_init(&own_full[i], 1), mbar_init(&own_empty[i], 1);
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < BUFS; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], Cfg::WARPS), mbar_init(&g_full[i], Cfg::WARPS), mbar_init(&g_empty[i], 1);
        mbar_init(o_full, 1);
        mbar_init(o_empty, Cfg::WARPS * GROUPS);
        mbar_init(drained, 2);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem, tmem_s = tmem + Cfg::O_COLS, tmem_g = tmem_s + BUFS * NB;

    if (warp == 0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::FEW_REGS));
        if (lane == 0) {
            uint32_t s = 0, parity = 1, fills = 0, owns = 0;
            bool live = true;
            for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
                const CeFusedUnit unit(a, u);
                const uint32_t o = owns % OWNS;
                if (!mbar_wait(&own_empty[o], ((owns / OWNS) & 1u) ^ 1u, s_abort, a.d_error)) break;
                mbar_expect_tx(&own_full[o], Cfg::OWN_BYTES);
                for (int k = 0; k < KB; ++k) tma_load_3d(base + o * Cfg::OWN_BYTES + k * (TG_M * 128), &tmOwn, &own_full[o], k * 64, unit.own0, 0);
                ++owns;
                for (int t = 0; t < unit.tiles; ++t) {
                    if (!mbar_wait(&empty[s], parity, s_abort, a.d_error)) { live = false; break; }
                    unsigned char* const column = s_columns + s * Cfg::COLUMNS * Cfg::COLUMN_BYTES;
                    mbar_expect_tx(&full[s], Cfg::STAGE_BYTES + (ROWS ? Cfg::COLUMNS : BIAS ? 1 : 0) * Cfg::COLUMN_BYTES);
                    if (ROWS) {
                        bulk_load(column, a.terms + (int64_t)unit.tile(t) * NB, Cfg::COLUMN_BYTES, &full[s]);
                        bulk_load(column + Cfg::COLUMN_BYTES, a.factors + (int64_t)unit.tile(t) * NB, Cfg::COLUMN_BYTES, &full[s]);
                        bulk_load(column + 2 * Cfg::COLUMN_BYTES, a.target_cols + (int64_t)unit.tile(t) * NB, Cfg::COLUMN_BYTES, &full[s]);
                    } else if (BIAS) {
                        bulk_load(column, a.bias + (int64_t)unit.tile(t) * NB, Cfg::COLUMN_BYTES, &full[s]);
                    }
                    for (int k = 0; k < KB; ++k)
                        tma_load_3d(s_other + s * Cfg::STAGE_BYTES + k * (NB * 128), &tmOther, &full[s], k * 64, unit.tile(t) * NB, 0);
                    ++fills;
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            s_fills[0] = fills;
            s_fills[1] = owns;
        }
    } else if (warp == 1) {  // first products
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::FEW_REGS));
        uint32_t n = 0, s = 0, s_parity = 0, owns = 0;
        bool live = true;
        for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
            const CeFusedUnit unit(a, u);
            const uint32_t o = owns % OWNS;
            if (!mbar_wait_warp(&own_full[o], (owns / OWNS) & 1u, s_abort, a.d_error)) break;
            ++owns;
            const uint64_t da = tg_desc<false>(smem_u32(base + o * Cfg::OWN_BYTES));
            for (int t = 0; t < unit.tiles; ++t, ++n) {
                const uint32_t b = n % BUFS;
                if (!mbar_wait_warp(&s_empty[b], ((n / BUFS) & 1u) ^ 1u, s_abort, a.d_error) || !mbar_wait_warp(&full[s], s_parity, s_abort, a.d_error)) {
                    live = false;
                    break;
                }
                tc_fence_after();
                const uint64_t db = tg_desc<false>(smem_u32(s_other + s * Cfg::STAGE_BYTES));
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        tc_mma_warp<false>(tmem_s + b * NB, da + k * (TG_M * 128 / 16) + j * 2, db + k * (NB * 128 / 16) + j * 2, a.idesc_s, (k | j) != 0);
                tc_commit_warp(&s_full[b]);
                if (t + 1 == unit.tiles) tc_commit_warp(&own_empty[o]);
                if (++s == STAGES) { s = 0; s_parity ^= 1u; }
            }
        }
    } else if (warp == 2) {  // second products
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::FEW_REGS));
        uint32_t n = 0, s = 0, units = 0;
        bool live = true;
        for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x, ++units) {
            const CeFusedUnit unit(a, u);
            if (!mbar_wait_warp(o_empty, (units & 1u) ^ 1u, s_abort, a.d_error)) break;
            for (int t = 0; t < unit.tiles; ++t, ++n) {
                const uint32_t b = n % BUFS;
                if (!mbar_wait_warp(&g_full[b], (n / BUFS) & 1u, s_abort, a.d_error)) { live = false; break; }
                tc_fence_after();
                const uint64_t db = tg_desc<false>(smem_u32(s_other + s * Cfg::STAGE_BYTES)) | ((uint64_t)((NB * 128) >> 4) << 16);
#pragma unroll
                for (int k = 0; k < NB / 16; ++k) tc_mma_ts_warp(tmem, tmem_g + b * (NB / 2) + k * 8, db + k * 128, a.idesc_o, (t | k) != 0);
                tc_commit_warp(&empty[s]);
                tc_commit_warp(&g_empty[b]);
                if (++s == STAGES) s = 0;
            }
            if (live) tc_commit_warp(o_full);
        }
    } else if (warp == 3) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::FEW_REGS));
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::MANY_REGS));
        constexpr int CW = Cfg::CW;
        const int quarter = warp & 3, group = (warp - 4) / Cfg::WARPS, col0 = (warp - 4) % Cfg::WARPS / 4 * CW;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        // dX in half precision: what brings the largest factor next to 2^15
        const int exponent = HALF && ROWS ? ce_scale_exponent(a.amax) : 0;
        const float up = ldexpf(1.f, exponent - CE_HALF_SHIFT);
        const uint64_t cc = f2_pack(a.c, a.c), up2 = f2_pack(up, up);
        bool live = true;
        uint32_t nth = 0, units = 0;
        for (unsigned u = blockIdx.x; u < a.units; u += gridDim.x, ++units) {
            const CeFusedUnit unit(a, u);
            const int first_own = unit.own0 + quarter * 32, mine = first_own + lane;
            const bool in = mine < a.own;
            float my_term = 0.f;  // of a query, or a row's bias
            int my_target = -1;
            if (in) {
                if (!ROWS) {
                    my_term = __ldcg(a.terms + mine);
                    my_target = __ldcg(a.target_cols + mine);
                } else if (BIAS) {
                    my_term = __ldcg(a.bias + mine);
                }
            }
            const uint64_t term2 = f2_pack(my_term, my_term);
            const int ahead = (int)((GROUPS + group - nth % GROUPS) % GROUPS);  // the group's first tile of the unit
            for (int t = ahead; t < unit.tiles; t += GROUPS) {
                const uint32_t n = nth + t, b = n % BUFS;
                const int first = unit.tile(t) * NB + col0;
                const float* const columns = reinterpret_cast<const float*>(s_columns + n % STAGES * (Cfg::COLUMNS * Cfg::COLUMN_BYTES)) + col0;
                const float* const factors = columns + NB;
                const int* const targets = reinterpret_cast<const int*>(factors + NB);
                if ((ROWS || BIAS) && live) live = mbar_wait_warp(&full[n % STAGES], (n / STAGES) & 1u, s_abort, a.d_error);
                // what is seldom: a target in the warp's part of the tile, the end of the other side
                bool seldom;
                if (ROWS) {
                    bool hit = false;
#pragma unroll
                    for (int i = 0; i < CW / 32; ++i) hit = hit || (unsigned)(targets[i * 32 + lane] - a.own0 - first_own) < 32u;
                    seldom = __any_sync(0xFFFFFFFFu, hit);
                } else {
                    seldom = a.other - first < CW || __any_sync(0xFFFFFFFFu, (unsigned)(my_target - first) < (unsigned)CW);
                }
                if (live) live = mbar_wait_warp(&s_full[b], (n / BUFS) & 1u, s_abort, a.d_error);
                tc_fence_after();
                const uint32_t from = tmem_s + lanes + b * NB + col0, to = tmem_g + lanes + b * (NB / 2) + col0 / 2;
                uint32_t r[CW / 32][32];
#pragma unroll
                for (int i = 0; i < CW / 32; ++i) tg_ld32(from + i * 32, r[i]);
                tc_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[b]);
                if (live) live = mbar_wait_warp(&g_empty[b], ((n / BUFS) & 1u) ^ 1u, s_abort, a.d_error);
                tc_fence_after();
                auto make = [&](auto checked) {
#pragma unroll
                    for (int i = 0; i < CW / 32; ++i) {
                        float v[32];
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            ulonglong2 x = make_ulonglong2(term2, term2);
                            if (ROWS || BIAS) x = *reinterpret_cast<const ulonglong2*>(columns + i * 32 + j);
                            // a row's bias, then the query's term
                            const bool own_first = ROWS && BIAS;
                            uint64_t t0 = f2_fma(f2_pack(__uint_as_float(r[i][j]), __uint_as_float(r[i][j + 1])), cc, own_first ? term2 : x.x);
                            uint64_t t1 = f2_fma(f2_pack(__uint_as_float(r[i][j + 2]), __uint_as_float(r[i][j + 3])), cc, own_first ? term2 : x.y);
                            if (BIAS) t0 = f2_add(t0, own_first ? x.x : term2), t1 = f2_add(t1, own_first ? x.y : term2);
                            f2_unpack(t0, v[j], v[j + 1]);
                            f2_unpack(t1, v[j + 2], v[j + 3]);
#pragma unroll
                            for (int k = j; k < j + 4; ++k) v[k] = ce_exp2(v[k]);
                            if (ROWS) {
                                ulonglong2 f = *reinterpret_cast<const ulonglong2*>(factors + i * 32 + j);
                                if (HALF) f = make_ulonglong2(f2_mul(f.x, up2), f2_mul(f.y, up2));
                                f2_unpack(f2_mul(f2_pack(v[j], v[j + 1]), f.x), v[j], v[j + 1]);
                                f2_unpack(f2_mul(f2_pack(v[j + 2], v[j + 3]), f.y), v[j + 2], v[j + 3]);
                            }
                        }
                        if (decltype(checked)::value) {
                            if (ROWS) {
                                const int target = targets[i * 32 + lane] - a.own0 - first_own;
                                unsigned hits = __ballot_sync(0xFFFFFFFFu, (unsigned)target < 32u), zero = 0;
                                while (hits) {  // columns whose target is one of the warp's rows
                                    const int j = __ffs(hits) - 1;
                                    hits &= hits - 1u;
                                    if (__shfl_sync(0xFFFFFFFFu, target, j) == lane) zero |= 1u << j;
                                }
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (zero >> j & 1u) v[j] = 0.f;
                            } else {
                                const int at = my_target - (first + i * 32), left = a.other - (first + i * 32);
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (j == at || j >= left) v[j] = 0.f;
                            }
                        }
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = pack_scores(static_cast<const T*>(nullptr), v[2 * j], v[2 * j + 1]);
                        if (decltype(checked)::value) __syncwarp();  // all lanes store together
                        tg_store16(to + i * 16, w);
                    }
                };
                if (seldom) make(std::true_type());
                else make(std::false_type());
                tg_store_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&g_full[b]);
            }
            nth += unit.tiles;
            // the sums, 32 columns to four warps in turn
            if (live) live = mbar_wait_warp(o_full, units & 1u, s_abort, a.d_error);
            tc_fence_after();
            const bool typed = ROWS && !a.parts;
            const bool wide = typed ? (a.d & 7) == 0 && (a.ld & 7) == 0 && ((uintptr_t)a.out & 15) == 0 : (a.d & 3) == 0;
#pragma unroll 1
            for (int c0 = (warp - 4) / 4 * 32; c0 < a.d; c0 += Cfg::WARPS * GROUPS / 4 * 32) {
                uint32_t r[32];
                tg_read(tmem + lanes + c0, live, r);
                float v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
                if (typed) {
                    const float scale = HALF ? ce_scale_back(a.inv_t, exponent) : a.inv_t;
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] *= scale;
                    ce_add_own(v, a.where + mine, a.where_stride, in ? a.own_splits : 0, a.sums, a.d, c0, a.inv_t);
                }
                T* const o = reinterpret_cast<T*>(a.out) + (int64_t)mine * a.ld + c0;
                float* const part = a.parts + ((int64_t)unit.block * a.own + mine) * a.d + c0;
                if (!wide) {
                    ce_turn(v, lane);
                    if (c0 + lane < a.d) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (first_own + j >= a.own) break;
                            if (typed) store_score(o + (int64_t)(j - lane) * a.ld + lane, v[j]);
                            else part[(int64_t)(j - lane) * a.d + lane] = v[j];
                        }
                    }
                } else if (in && typed) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        if (c0 + j >= a.d) break;
                        const T* const t = nullptr;
                        *reinterpret_cast<uint4*>(o + j) =
                            make_uint4(pack_scores(t, v[j], v[j + 1]), pack_scores(t, v[j + 2], v[j + 3]), pack_scores(t, v[j + 4], v[j + 5]), pack_scores(t, v[j + 6], v[j + 7]));
                    }
                } else if (in) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (c0 + j >= a.d) break;
                        *reinterpret_cast<float4*>(part + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*s_abort) {  // all roles are done: what they issued may not be
        if (threadIdx.x == 0) {
            mbar_wait_landed(full, STAGES, s_fills[0]);
            mbar_wait_landed(own_full, OWNS, s_fills[1]);
        }
        if (warp == 1 || warp == 2) {
            tc_commit_warp(drained);
            mbar_wait_landed(drained, 1, 1);
        }
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
template <int KB, bool ROWS, bool BIAS, bool HALF>
inline void ce_fused_launch(const CtxPtr& c, const CUtensorMap& own, const CUtensorMap& other, const CeFusedArgs& a, cudaStream_t stream) {
    using Cfg = CeFusedCfg<KB>;
    static thread_local uint64_t ready = 0;  // devices whose limit is set
    if (c->device >= 64 || !(ready >> c->device & 1)) {
        cudaFuncAttributes is;
        CU_CHECK(cudaFuncGetAttributes(&is, ce_fused_kernel<KB, ROWS, BIAS, HALF>));
        if (is.numRegs != Cfg::REGS) fail(CULSH_ERR_INTERNAL, "built with %d registers a thread in place of %d", is.numRegs, Cfg::REGS);  // the warps' shares would not add up
        CU_CHECK(cudaFuncSetAttribute(ce_fused_kernel<KB, ROWS, BIAS, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        if (c->device < 64) ready |= 1ull << c->device;
    }
    launch_next(stream, ce_fused_kernel<KB, ROWS, BIAS, HALF>, std::min<unsigned>(a.units, (unsigned)c->sm_count), (unsigned)Cfg::THREADS, (size_t)Cfg::SMEM, own, other, a);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
