// Gradient of the cross entropy for rows of up to 256 values of 16 bits: G does not leave the SM.
//
// A CTA keeps 128 entries of one side ("own": rows for dX, queries for dQ) and goes through the other, a tile at a time:  S = own . other^T into tensor memory,  G = factor exp2(c S + term)
// by the epilogue's threads and back into tensor memory as 16 bits, on top of S,  O += G . other with G as the operand that lies in tensor memory.  The other side's tile is loaded once for
// both products: K along its rows for the first, across them for the second.  S is made again for the other gradient: 8 m n d operations in place of 6, against 6 bytes of G written and read
// for each of the m n entries.
//
// One warp loads, one issues the MMAs, groups of four warps take the tiles in turn, one for each buffer of S.  The second product of a tile is issued BUFS - 1 tiles behind its first, so that
// neither waits for the exponentials.  Sums of more than 32,768 entries are split (the accumulators cut off, see tc_gemm.cuh), those of dQ over units, whose sums ce_finish_kernel adds up.
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

// What a power of two brings the largest factor to [2^14, 2^15].
__device__ __forceinline__ int ce_scale_exponent(const uint32_t* amax) {
    const uint32_t bits = amax ? __ldcg(amax) : 0u;
    return bits == 0u ? 0 : min(max(14 + 127 - (int)(bits >> 23), -100), 100);
}

struct CeFusedArgs {
    int* d_error;
    unsigned units;
    uint32_t idesc_s, idesc_o;
    int own, other;           // entries of either side
    int tiles_own, tiles_other, block;
    int d;
    float c;
    const float* bias;        // of the rows, in powers of two, or NULL
    const float* terms;       // of the queries
    const float* factors;
    const uint32_t* amax;
    const int* target_cols;
    float* parts;             // dQ: [block][query][d]
    void* out;                // dX
    int64_t ld;
    const int* where;
    const float* sums;
    float inv_t;
};

// KB: boxes of 64 values in a row.
template <int KB>
struct CeFusedCfg {
    static constexpr int NB = KB == 4 ? 64 : 128;             // entries of a tile of the other side
    static constexpr int O_COLS = KB * 64, BUFS = KB == 4 ? 4 : 3, GROUPS = BUFS;
    static constexpr int OWN_BYTES = KB * TG_M * 128, OWNS = KB == 4 ? 1 : 2;
    static constexpr int STAGE_BYTES = KB * NB * 128, STAGES = KB == 1 ? 8 : 4;
    static constexpr int THREADS = 64 + 128 * GROUPS;
    static constexpr int COLUMN_BYTES = GROUPS * 4 * NB * 8;
    static constexpr int SMEM = OWNS * OWN_BYTES + STAGES * STAGE_BYTES + COLUMN_BYTES + 1024 /*barriers*/ + 1024 /*alignment slack*/;
    static_assert(O_COLS + BUFS * NB <= 512 && SMEM <= 227 * 1024 && STAGES >= BUFS, "");
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

struct CeFusedUnit {
    int own0, tile0, tiles, block;
    __device__ __forceinline__ CeFusedUnit(const CeFusedArgs& a, unsigned u) {
        block = (int)(u / (unsigned)a.tiles_own);
        own0 = (int)(u - (unsigned)block * a.tiles_own) * TG_M;
        tile0 = block * a.block;
        tiles = min(a.block, a.tiles_other - tile0);
    }
};

// What the columns of a tile bring, for one warp: lane i of a warp has columns i, i + 32 ...  ROWS (own: rows, columns: queries): term, factor and target; else the rows' bias.
template <int NB, bool ROWS, bool BIAS, bool HALF>
struct CeColumns {
    float term[NB / 32], factor[NB / 32];
    int target[NB / 32];
    __device__ __forceinline__ void fetch(const CeFusedArgs& a, int first, int end, int lane) {
#pragma unroll
        for (int i = 0; i < NB / 32; ++i) {
            const int j = first + i * 32 + lane;
            const bool in = j < end;
            if (ROWS) {
                term[i] = in ? __ldcg(a.terms + j) : -INFINITY;  // no entry: 0, whatever the bias
                factor[i] = in ? __ldcg(a.factors + j) : 0.f;
                target[i] = in ? __ldcg(a.target_cols + j) : -1;
            } else if (BIAS) {
                term[i] = in ? __ldcg(a.bias + j) : 0.f;
            }
        }
    }
    __device__ __forceinline__ void put(float* s, int exponent, int lane) const {
        if (!ROWS && !BIAS) return;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NB / 32; ++i) {
            s[i * 32 + lane] = term[i];
            if (ROWS) s[NB + i * 32 + lane] = HALF ? ldexpf(factor[i], exponent) : factor[i];
        }
        __syncwarp();
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
    float* const s_columns = reinterpret_cast<float*>(s_other + STAGES * Cfg::STAGE_BYTES);
    uint64_t* const own_full = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(s_columns) + Cfg::COLUMN_BYTES);
    uint64_t* const own_empty = own_full + OWNS;
    uint64_t* const full = own_empty + OWNS;
    uint64_t* const empty = full + STAGES;
    uint64_t* const s_full = empty + STAGES;   // S is there
    uint64_t* const s_empty = s_full + BUFS;   // and its place free again
    uint64_t* const g_full = s_empty + BUFS;   // G is there
    uint64_t* const o_full = g_full + BUFS;
    uint64_t* const o_empty = o_full + 1;
    uint64_t* const drained = o_empty + 1;
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    uint32_t* const s_fills = s_tmem + 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < OWNS; ++i) mbar_init(&own_full[i], 1), mbar_init(&own_empty[i], 1);
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < BUFS; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 1), mbar_init(&g_full[i], 4);
        mbar_init(o_full, 1);
        mbar_init(o_empty, 4 * GROUPS);
        mbar_init(drained, 1);
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
    const uint32_t tmem = *s_tmem, tmem_s = tmem + Cfg::O_COLS;

    if (warp == 0) {
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
                    mbar_expect_tx(&full[s], Cfg::STAGE_BYTES);
                    for (int k = 0; k < KB; ++k)
                        tma_load_3d(s_other + s * Cfg::STAGE_BYTES + k * (NB * 128), &tmOther, &full[s], k * 64, (unit.tile0 + t) * NB, 0);
                    ++fills;
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            s_fills[0] = fills;
            s_fills[1] = owns;
        }
    } else if (warp == 1) {
        constexpr int LAG = BUFS - 1;
        // The second products follow the first ones by LAG tiles: where they are in the units.
        uint32_t n1 = 0, n2 = 0, owns = 0, units2 = 0;  // tiles, units
        unsigned u2 = blockIdx.x;
        int t2 = 0, tiles2 = u2 < a.units ? CeFusedUnit(a, u2).tiles : 0;
        bool live = true;
        auto second = [&]() {
            const uint32_t b = n2 % BUFS, s = n2 % STAGES;
            if (t2 == 0 && !mbar_wait_warp(o_empty, (units2 & 1u) ^ 1u, s_abort, a.d_error)) return false;
            if (!mbar_wait_warp(&g_full[b], (n2 / BUFS) & 1u, s_abort, a.d_error)) return false;
            tc_fence_after();
            const uint64_t db = tg_desc<false>(smem_u32(s_other + s * Cfg::STAGE_BYTES)) | ((uint64_t)((NB * 128) >> 4) << 16);
#pragma unroll
            for (int i = 0; i < NB / 16; ++i) tc_mma_ts_warp(tmem, tmem_s + b * NB + i * 8, db + i * 128, a.idesc_o, (t2 | i) != 0);
            tc_commit_warp(&empty[s]);
            tc_commit_warp(&s_empty[b]);
            ++n2;
            if (++t2 == tiles2) {
                tc_commit_warp(o_full);
                ++units2;
                t2 = 0;
                u2 += gridDim.x;
                tiles2 = u2 < a.units ? CeFusedUnit(a, u2).tiles : 0;
            }
            return true;
        };
        for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
            const CeFusedUnit unit(a, u);
            const uint32_t o = owns % OWNS;
            if (!mbar_wait_warp(&own_full[o], (owns / OWNS) & 1u, s_abort, a.d_error)) { live = false; break; }
            ++owns;
            const uint64_t da = tg_desc<false>(smem_u32(base + o * Cfg::OWN_BYTES));
            for (int t = 0; t < unit.tiles; ++t, ++n1) {
                const uint32_t b = n1 % BUFS, s = n1 % STAGES;
                if (!mbar_wait_warp(&s_empty[b], ((n1 / BUFS) & 1u) ^ 1u, s_abort, a.d_error) || !mbar_wait_warp(&full[s], (n1 / STAGES) & 1u, s_abort, a.d_error)) {
                    live = false;
                    break;
                }
                tc_fence_after();
                const uint64_t db = tg_desc<false>(smem_u32(s_other + s * Cfg::STAGE_BYTES));
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tc_mma_warp<false>(tmem_s + b * NB, da + k * (TG_M * 128 / 16) + i * 2, db + k * (NB * 128 / 16) + i * 2, a.idesc_s, (k | i) != 0);
                tc_commit_warp(&s_full[b]);
                if (t + 1 == unit.tiles) tc_commit_warp(&own_empty[o]);
                if (n1 >= LAG && !second()) { live = false; break; }
            }
        }
        while (live && n2 < n1) live = second();
    } else {
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        float* const columns = s_columns + (warp - 2) * (2 * NB);
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const int exponent = HALF ? ce_scale_exponent(a.amax) : 0;
        bool live = true;
        uint32_t nth = 0, units = 0;
        for (unsigned u = blockIdx.x; u < a.units; u += gridDim.x, ++units) {
            const CeFusedUnit unit(a, u);
            const int first_own = unit.own0 + quarter * 32, mine = first_own + lane;
            const bool in = mine < a.own;
            float my_term = 0.f, my_factor = 0.f;
            int my_target = -1;
            if (!ROWS && in) {
                my_term = __ldcg(a.terms + mine);
                my_factor = __ldcg(a.factors + mine);
                if (HALF) my_factor = ldexpf(my_factor, exponent);
                my_target = __ldcg(a.target_cols + mine);
            }
            if (ROWS && BIAS && in) my_term = __ldcg(a.bias + mine);
            CeColumns<NB, ROWS, BIAS, HALF> next;
            const int ahead = (int)((GROUPS + group - nth % GROUPS) % GROUPS);  // the group's first tile of the unit
            if (ahead < unit.tiles) next.fetch(a, (unit.tile0 + ahead) * NB, a.other, lane);
            for (int t = ahead; t < unit.tiles; t += GROUPS) {
                const uint32_t n = nth + t, b = n % BUFS;
                const int first = (unit.tile0 + t) * NB;
                int target[NB / 32];
                if (ROWS) {
#pragma unroll
                    for (int i = 0; i < NB / 32; ++i) target[i] = next.target[i] - first_own;
                }
                next.put(columns, exponent, lane);
                if (t + GROUPS < unit.tiles) next.fetch(a, first + GROUPS * NB, a.other, lane);
                if (live) live = mbar_wait_warp(&s_full[b], (n / BUFS) & 1u, s_abort, a.d_error);
                tc_fence_after();
                const uint32_t place = tmem_s + lanes + b * NB;
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += 32) {
                    uint32_t r[32];
                    tc_ld32(place + c0, r);
                    tc_ld_wait();
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float s = __uint_as_float(r[j]);
                        if (ROWS) v[j] = ce_exp2(fmaf(s, a.c, BIAS ? columns[c0 + j] + my_term : columns[c0 + j])) * columns[NB + c0 + j];
                        else v[j] = ce_exp2(fmaf(s, a.c, BIAS ? my_term + columns[c0 + j] : my_term)) * my_factor;
                    }
                    if (ROWS) {
                        unsigned hits = __ballot_sync(0xFFFFFFFFu, (unsigned)target[c0 / 32] < 32u);
                        if (hits) {  // columns whose target is one of the warp's rows
                            unsigned zero = 0;
                            while (hits) {
                                const int j = __ffs(hits) - 1;
                                hits &= hits - 1u;
                                if (__shfl_sync(0xFFFFFFFFu, target[c0 / 32], j) == lane) zero |= 1u << j;
                            }
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (zero >> j & 1u) v[j] = 0.f;
                        }
                    } else {
                        const int at = my_target - (first + c0), left = a.other - (first + c0);
                        if (left < 32 || __any_sync(0xFFFFFFFFu, (unsigned)at < 32u)) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j == at || j >= left) v[j] = 0.f;
                        }
                    }
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) w[j] = pack_scores(static_cast<const T*>(nullptr), v[2 * j], v[2 * j + 1]);
                    tg_store16(place + c0 / 2, w);
                }
                tg_store_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&g_full[b]);
            }
            nth += unit.tiles;
            // the sums, 32 columns to a group in turn
            if (live) live = mbar_wait_warp(o_full, units & 1u, s_abort, a.d_error);
            tc_fence_after();
            int slot = -1;
            if (ROWS && in) slot = __ldcg(a.where + mine);
            const bool wide = ROWS ? (a.d & 7) == 0 && (a.ld & 7) == 0 && ((uintptr_t)a.out & 15) == 0 : (a.d & 3) == 0;
#pragma unroll 1
            for (int c0 = group * 32; c0 < a.d; c0 += GROUPS * 32) {
                uint32_t r[32];
                tg_read(tmem + lanes + c0, live, r);
                if (!in) continue;
                if constexpr (ROWS) {
                    const float scale = a.inv_t;
                    T* const o = reinterpret_cast<T*>(a.out) + (int64_t)mine * a.ld + c0;
                    const float* const extra = a.sums + (int64_t)slot * a.d + c0;
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        v[j] = __uint_as_float(r[j]);
                        if (HALF) v[j] = ldexpf(v[j], -exponent);
                        if (slot >= 0 && c0 + j < a.d) v[j] += __ldcg(extra + j);
                        v[j] *= scale;
                    }
                    if (wide) {
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            if (c0 + j >= a.d) break;
                            const T* const t = nullptr;
                            *reinterpret_cast<uint4*>(o + j) = make_uint4(pack_scores(t, v[j], v[j + 1]), pack_scores(t, v[j + 2], v[j + 3]), pack_scores(t, v[j + 4], v[j + 5]),
                                                                          pack_scores(t, v[j + 6], v[j + 7]));
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c0 + j < a.d) store_score(o + j, v[j]);
                    }
                } else {
                    float* const o = a.parts + ((int64_t)unit.block * a.own + mine) * a.d + c0;
                    if (wide) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            if (c0 + j >= a.d) break;
                            *reinterpret_cast<uint4*>(o + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c0 + j < a.d) o[j] = __uint_as_float(r[j]);
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
        if (warp == 1) {
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
        CU_CHECK(cudaFuncSetAttribute(ce_fused_kernel<KB, ROWS, BIAS, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        if (c->device < 64) ready |= 1ull << c->device;
    }
    launch_next(stream, ce_fused_kernel<KB, ROWS, BIAS, HALF>, std::min<unsigned>(a.units, (unsigned)c->sm_count), (unsigned)Cfg::THREADS, (size_t)Cfg::SMEM, own, other, a);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
