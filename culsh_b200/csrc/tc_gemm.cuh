// Matrix products on the 5th-generation tensor cores, with what is done to a tile of them left to a policy: 16-bit floats (tcgen05.mma kind::f16, fp32
// accumulators) and 8-bit integers (kind::i8, int32 accumulators, exact).
//
// Persistent CTAs with a warp for the TMA loads, one for the MMAs and eight or sixteen of epilogue, in groups of four, which take the tiles in turn or a part of a tile's columns each: a
// warp of a group reads its quarter of the accumulator's 128 lanes.  A tile is 128 entries of the M side by up to P::BN of the N side; a stage holds 128 bytes of K for both.  Two CTAs can
// work as a pair (PAIR) on 256 entries of the M side: each loads its 128 and half of the N side, which the MMAs, issued by the first of the two, read from both (cta_group::2): two thirds of the
// bytes from L2 and of the reads of shared memory.  Either
// operand may lie with K or with the other side along its rows ("MN-major"): both are loaded in boxes of 128 bytes by so many rows, swizzled over 128 bytes, and
// only the descriptors differ.  Operands that are held as sums of planes (32-bit floats as three bfloat16) are multiplied pair by pair, the small ones first, so that the
// accumulator is small while they come.  Every wait is bounded (mbar_wait); a CTA whose wait ran out records it, its tiles are NaN, and it waits for what it has in flight
// before it gives its memory back.  No load uses cluster multicast.
//
// The accumulators cut off what their adds leave behind 32 bits, half a unit each time on average and always to the same side: 128 adds (K of 2,048) leave a sum 4e-6 of it too small.  A
// policy may have K taken in segments of so many steps, each in an accumulator of its own, which its epilogue adds up.
//
// A policy has:  Args with `units` and `d_error`;  Unit(args, u) with `tiles`, `k0`, `k1` (steps of K);  load(), which brings a step of a tile (rank: which
// of a pair's CTAs);  n_mma(args, unit, tile), columns of a tile;  EPI_WARPS;  PARTS, whether the groups share a tile;  SEGMENTS, whether K may be taken in them, of Args'
// `segment` steps;  Epilogue with unit_begin(), segment() of all accumulators of a tile but the last, tile() and unit_end().
#pragma once

#include "tc_ptx.cuh"
#include "mx_product.cuh"

namespace culsh_b200 {

constexpr int TG_M = 128, TG_SMEM = 224 * 1024;
constexpr int TG_BOX_BYTES = 8192;  // of an MN-major operand: 64 entries by 64 of K

// Pairs of planes, in the order in which they are multiplied.  Of three planes each: what is left out is below 2^-24 of the product.
template <int PLANES>
struct PlanePairs;
template <>
struct PlanePairs<1> {
    static constexpr int N = 1;
    static __device__ __forceinline__ int a(int) { return 0; }
    static __device__ __forceinline__ int b(int) { return 0; }
};
template <>
struct PlanePairs<3> {  // (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
    static constexpr int N = 6;
    static __device__ __forceinline__ int a(int p) { return p == 0 ? 2 : p == 2 || p == 3 ? 1 : 0; }
    static __device__ __forceinline__ int b(int p) { return p == 1 ? 2 : p == 2 || p == 4 ? 1 : 0; }
};

// PAIR: the barrier is the first CTA's of the two.
template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(smem_u32(smem_dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(smem_u32(smem_dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    tma_load_3d<false>(smem_dst, map, smem_u32(bar), x, y, z);
}
#define TG_MMA(GROUP, KIND)                                                                          \
    asm volatile(                                                                                     \
        "{\n\t.reg .pred p, e;\n\t"                                                                  \
        "elect.sync _|e, 0xFFFFFFFF;\n\t"                                                             \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                   \
        "@e tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}"                \
        ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                                    \
        : "memory")
template <bool I8, bool PAIR = false>
__device__ __forceinline__ void tc_mma_warp(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (I8 && PAIR) TG_MMA("2", "i8");
    else if constexpr (I8) TG_MMA("1", "i8");
    else if constexpr (PAIR) TG_MMA("2", "f16");
    else TG_MMA("1", "f16");
}
#undef TG_MMA
// The barrier at the same place of both CTAs of a pair.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xFFFFFFFF;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(smem_u32(bar)), "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ uint32_t first_of_pair(const void* p) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(p)));
    return at;
}
// For what has been read of tensor memory, which tcgen05.fence orders; an arrival that releases writes to the whole cluster waits for all of the warp's memory operations.
__device__ __forceinline__ void mbar_arrive_at(uint32_t at) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(at) : "memory"); }
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// K along the rows: groups of 8 rows of 128 bytes one behind the other.  Else: rows of 64 entries, one for each of K; groups of 8 rows, and boxes for the next 64 entries.
template <bool MN>
__device__ __forceinline__ uint64_t tg_desc(uint32_t saddr) {
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | (MN ? (uint64_t)(TG_BOX_BYTES >> 4) << 16 : 0ull) | ((saddr & 0x3FFFFu) >> 4);
}
enum TgType : int { TG_F16 = 0, TG_BF16 = 1, TG_I8 = 2 };
// Both operands of one type: float accumulators, or int32 of signed 8-bit integers.
inline uint32_t tg_idesc(TgType t, bool a_mn, bool b_mn) {
    const uint32_t type = t == TG_F16 ? 0u : 1u;
    return ((t == TG_I8 ? 2u : 1u) << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
}

template <typename P>
__device__ __forceinline__ int tg_segments(const typename P::Args& a, const typename P::Unit& u) {
    if constexpr (P::SEGMENTS) return (u.k1 - u.k0 + a.segment - 1) / a.segment;
    else return 1;
}
// Steps of a segment: first and last.
template <typename P>
__device__ __forceinline__ int2 tg_segment(const typename P::Args& a, const typename P::Unit& u, int nth) {
    if constexpr (P::SEGMENTS) return make_int2(u.k0 + nth * a.segment, min(u.k1, u.k0 + (nth + 1) * a.segment));
    else return make_int2(u.k0, u.k1);
}

template <typename P>
struct TgCfg {
    static constexpr int A_BYTES = TG_M * 128, B_ROWS = P::BN / (P::PAIR ? 2 : 1), B_BYTES = B_ROWS * 128, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = (TG_SMEM - P::EPI_BYTES) / STAGE_BYTES;
    static constexpr int ACCS = 512 / P::BN, GROUPS = P::EPI_WARPS / 4, THREADS = 64 + 32 * P::EPI_WARPS;
    static constexpr int SMEM = STAGES * STAGE_BYTES + P::EPI_BYTES + 1024 /*barriers*/ + 1024 /*alignment slack*/;
    static constexpr uint32_t M_BITS = (uint32_t)((P::PAIR ? 2 * TG_M : TG_M) >> 4) << 24;
    static_assert(STAGES >= 2 && (2 * STAGES + 2 * ACCS + 1) * 8 + 16 <= 1024 && SMEM <= 227 * 1024 && (P::PARTS || ACCS % GROUPS == 0), "");
};

template <typename P>
__global__ void __launch_bounds__(TgCfg<P>::THREADS, 1)
tc_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, typename P::Args a, KernelBefore before) {
    behind_kernel_before(before);
    using Cfg = TgCfg<P>;
    constexpr int STAGES = Cfg::STAGES, ACCS = Cfg::ACCS;
    constexpr bool PAIR = P::PAIR;
    extern __shared__ unsigned char tg_smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tg_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* s_epi = base + (size_t)STAGES * Cfg::STAGE_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_epi + P::EPI_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + ACCS;
    uint64_t* drained = acc_empty + ACCS;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    uint32_t* s_fills = s_tmem + 2;  // stages that have been loaded
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a pair takes a unit; its first CTA issues the MMAs, and has the barriers that loads and epilogues of both arrive at
    const unsigned rank = PAIR ? blockIdx.x & 1u : 0u, first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < ACCS; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], (P::PARTS ? P::EPI_WARPS : 4) * (PAIR ? 2 : 1));
        }
        mbar_init(drained, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) pair_sync();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, parity = 1, fills = 0;
            bool live = true;
            for (unsigned u = first; u < a.units && live; u += step) {
                const typename P::Unit unit(a, u);
                const int segments = tg_segments<P>(a, unit);
                for (int at = 0; at < unit.tiles * segments && live; ++at) {
                    const int t = at / segments;
                    const int2 steps = tg_segment<P>(a, unit, at - t * segments);
                    for (int pair = 0; pair < P::Pairs::N && live; ++pair) {
                        for (int k = steps.x; k < steps.y; ++k) {
                            if (!mbar_wait(&empty[s], parity, s_abort, a.d_error)) { live = false; break; }
                            unsigned char* st = base + (size_t)s * Cfg::STAGE_BYTES;
                            if (rank == 0) mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * Cfg::STAGE_BYTES);
                            P::load(a, unit, t, P::Pairs::a(pair), P::Pairs::b(pair), k, &tmA, &tmB, st, st + Cfg::A_BYTES, PAIR ? first_of_pair(&full[s]) : smem_u32(&full[s]),
                                    (int)rank);
                            ++fills;
                            if (++s == STAGES) { s = 0; parity ^= 1u; }
                        }
                    }
                }
            }
            *s_fills = fills;
        }
    } else if (warp == 1) {
        uint32_t s = 0, parity = 0, ab = 0, acc_parity = 1;
        bool live = rank == 0;
        for (unsigned u = first; u < a.units && live; u += step) {
            const typename P::Unit unit(a, u);
            const int segments = tg_segments<P>(a, unit);
            for (int at = 0; at < unit.tiles * segments && live; ++at) {
                const int t = at / segments;
                const int2 range = tg_segment<P>(a, unit, at - t * segments);
                if (!mbar_wait_warp(&acc_empty[ab], acc_parity, s_abort, a.d_error)) { live = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem + ab * P::BN;
                const uint32_t idesc = a.idesc | Cfg::M_BITS | ((uint32_t)((PAIR ? P::BN : P::n_mma(a, unit, t)) >> 3) << 17);  // a pair's CTAs hold half of N each, whatever is used of it
                const int steps = (range.y - range.x) * P::Pairs::N;
                for (int k = 0; k < steps; ++k) {
                    if (!mbar_wait_warp(&full[s], parity, s_abort, a.d_error)) { live = false; break; }
                    tc_fence_after();
                    const uint32_t st = smem_u32(base + (size_t)s * Cfg::STAGE_BYTES);
                    const uint64_t da = tg_desc<P::A_MN>(st), db = tg_desc<P::B_MN>(st + Cfg::A_BYTES);
#pragma unroll
                    for (int i = 0; i < 4; ++i)  // 32 bytes of K, or 16 rows of it
                        tc_mma_warp<P::I8, PAIR>(d_tmem, da + i * (P::A_MN ? 128 : 2), db + i * (P::B_MN ? 128 : 2), idesc, (k | i) != 0);
                    if (PAIR) tc_commit_pair(&empty[s]);
                    else tc_commit_warp(&empty[s]);
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
                if (live) {
                    if (PAIR) tc_commit_pair(&acc_full[ab]);
                    else tc_commit_warp(&acc_full[ab]);
                }
                if (++ab == ACCS) { ab = 0; acc_parity ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        typename P::Epilogue epi(a, s_epi, warp - 2, quarter, group, lane, (int)rank);
        bool live = true;
        uint32_t nth = 0;  // accumulator of the CTA
        for (unsigned u = first; u < a.units; u += step) {
            const typename P::Unit unit(a, u);
            const int segments = tg_segments<P>(a, unit);
            epi.unit_begin(a, unit);
            for (int t = 0; t < unit.tiles; ++t) {
                for (int g = 0; g < segments; ++g, ++nth) {
                    if (!P::PARTS && (int)(nth % Cfg::GROUPS) != group) continue;
                    const uint32_t ab = nth % ACCS, taddr = tmem + ((uint32_t)(quarter * 32) << 16) + ab * P::BN + (P::PARTS ? group * (P::BN / Cfg::GROUPS) : 0);
                    if (live) live = mbar_wait_warp(&acc_full[ab], (nth / ACCS) & 1u, s_abort, a.d_error);
                    tc_fence_after();
                    auto done = [&] {  // the accumulator has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (PAIR) mbar_arrive_at(first_of_pair(&acc_empty[ab]));
                            else mbar_arrive(&acc_empty[ab]);
                        }
                    };
                    if (P::SEGMENTS && g + 1 < segments) {
                        if constexpr (P::SEGMENTS) epi.segment(a, g == 0, taddr, live);
                        done();
                    } else {
                        epi.tile(a, unit, t, taddr, live, segments > 1, done);
                    }
                }
            }
            epi.unit_end(a, unit);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*s_abort) {  // all roles are done: what they issued may not be
        if (threadIdx.x == 0 && rank == 0) mbar_wait_landed(full, STAGES, *s_fills);
        if (warp == 1 && rank == 0) {
            if (PAIR) tc_commit_pair(drained);
            else tc_commit_warp(drained);
            mbar_wait_landed(drained, 1, 1);
        }
        __syncthreads();
    }
    if (PAIR) pair_sync();  // neither goes while the other may still arrive at its barriers, or read its half
    if (warp == 1) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Two floats in a register pair.
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

// Columns of an accumulator.  These instructions want all 32 lanes at the same place, and what stands in front may have let some go their own way (rows behind the last one are not stored).
__device__ __forceinline__ void tg_ld16(uint32_t taddr, uint32_t* r) {
    __syncwarp();
    tc_ld16(taddr, r);
}
__device__ __forceinline__ void tg_ld32(uint32_t taddr, uint32_t* r) {
    __syncwarp();
    tc_ld32(taddr, r);
}
__device__ __forceinline__ void tg_ld64(uint32_t taddr, uint32_t (&r)[2][32]) {
    tg_ld32(taddr, r[0]);
    tg_ld32(taddr + 32, r[1]);
}
// 32 of them, NaN where a wait ran out.
__device__ __forceinline__ void tg_read(uint32_t taddr, bool live, uint32_t (&r)[32]) {
    if (live) {  // the same for the warp
        tg_ld32(taddr, r);
        tc_ld_wait();
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = 0x7FFFFFFFu;
    }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
// `planes` matrices of rows x cols entries, rows `ld` entries apart, loaded 128 bytes by box_rows at a time; zeros behind every end.
inline CUtensorMap tg_map(const void* p, TgType type, int64_t rows, int64_t cols, int64_t ld, int planes, int64_t plane_bytes, int box_rows) {
    CUtensorMap m;
    PFN_encodeTiled enc = get_encode_tiled();
    const int size = type == TG_I8 ? 1 : 2;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    cuuint64_t strides[2] = {(cuuint64_t)(ld * size), (cuuint64_t)(planes > 1 ? plane_bytes : ld * size)};
    cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType t = type == TG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : type == TG_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    if (!enc || enc(&m, t, 3, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        fail(CULSH_ERR_CUDA, "no tensor map for %lld rows of %lld entries", (long long)rows, (long long)cols);
    return m;
}

template <typename P>
inline void tc_gemm(const CtxPtr& c, const CUtensorMap& ta, const CUtensorMap& tb, const typename P::Args& a, cudaStream_t stream) {
    using Cfg = TgCfg<P>;
    static thread_local uint64_t ready = 0;  // devices whose limit is set
    if (c->device >= 64 || !(ready >> c->device & 1)) {
        CU_CHECK(cudaFuncSetAttribute(tc_gemm_kernel<P>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        if (c->device < 64) ready |= 1ull << c->device;
    }
    const unsigned size = (unsigned)Cfg::SMEM, threads = (unsigned)Cfg::THREADS;
    if (P::PAIR) {
        launch_cluster(stream, tc_gemm_kernel<P>, 2 * std::min<unsigned>(a.units, (unsigned)c->sm_count / 2), 2u, threads, (size_t)size, ta, tb, a);
    } else {
        launch_next(stream, tc_gemm_kernel<P>, std::min<unsigned>(a.units, (unsigned)c->sm_count), threads, (size_t)size, ta, tb, a);
        KERNEL_CHECK();
    }
}

}  // namespace culsh_b200
