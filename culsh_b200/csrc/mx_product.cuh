// Scores of queries against all rows, both in microscaled 4-bit floating point (mx_rows.cuh): out[q][row] = sum_k q^_k x^_k, or the cosine, or the
// negative squared distance, on the 5th-generation tensor cores (tcgen05.mma kind::mxf4 with block scales, fp32 accumulators in tensor memory).
//
// Either side can be the M side of the MMA, whose 128 entries are the accumulator's lanes:
//   few queries (up to 64): the rows, so that no lane is idle, and a warp's store of a query is 32 neighbouring scores;
//   more: the queries, so that a lane holds neighbouring scores of a query, which it packs into 16 bytes.  They go through shared memory, from where sixteen lanes store
//   256 bytes of a query side by side.  (Stores by TMA were slower: 1,000 x 1M float32 scores 992 us against 792.)
// Codes come by TMA, swizzled; scale tiles of 512 bytes (128 rows by 4 blocks) lie in memory as the tensor cores
// take them and go from shared into tensor memory by tcgen05.cp, issued by the warp that issues the MMAs, in front of the two MMAs (64 values each) that read them.
//
// Persistent CTAs with a warp for the TMA loads, one for the MMAs and four, eight or twelve of epilogue; accumulators in turn.  Every wait is bounded
// (mbar_wait); a CTA whose wait ran out records it, fills what it has not done with NaN, and waits, with the same bound, for what it has in flight before it gives its memory back.  No load
// uses cluster multicast.
#pragma once

#include <algorithm>

#include "mx_rows.cuh"
#include "tc_ptx.cuh"

namespace culsh_b200 {

enum MxMetric : int { MX_DOT = 0, MX_COSINE = 1, MX_EUCLIDEAN = 2 };

constexpr int MXP_B = 128;  // entries of either side in a unit
constexpr int MXP_OUT_BYTES = 8192;  // 32 queries by 256 bytes

// More than 64 queries; the same of 1,024 values and more; up to 64; up to 16.
// With more queries, loads in flight and warps of epilogue share the SM: short rows wait for the scores to be stored (1,000 x 1M x 128 cosines: twelve warps 432 us, eight 507), long ones
// for their loads and MMAs in turn, no unit above 37 % (4,099 x 32,771 x 2,048: twelve warps and 102 KB of stages 244 us, eight and 136 KB 211, four and 170 KB 203).  The scores of 1,000 x 1M x 128 are written at 4.5 TB/s in bfloat16 and
// 5.3 in float32 (a fill of the memory: 3.9).  The fewer queries there are, the shorter is a unit, and the less of it the issuing warps and the epilogue can overlap: few queries have
// two or four CTAs on an SM, which share its tensor memory (one query, 1M x 128 rows: one CTA with eight warps of epilogue 38 us, four 21; 11.6 at the copy's rate).
enum MxpKind { MXP_MANY, MXP_LONG, MXP_FEW, MXP_FEWEST };
constexpr int MXP_FEW_MAX = 64, MXP_FEWEST_MAX = 16, MXP_LONG_GROUPS = 8;

// SPAN: bytes of a row in a stage, the swizzle span: 64 (one group) or 128 (two; of a row with an odd number of them the last stage has one, and zeros).
template <int SPAN, MxpKind KIND>
struct MxpCfg {
    static constexpr bool FEW = KIND == MXP_FEW || KIND == MXP_FEWEST;
    static constexpr int CTAS = !FEW ? 1 : KIND == MXP_FEW ? 2 : 4;
    static constexpr int GROUPS = SPAN / 64;
    static constexpr int A_BYTES = MXP_B * SPAN, S_BYTES = GROUPS * MX_TILE_BYTES;
    static constexpr int B_BYTES = (!FEW ? MXP_B : KIND == MXP_FEW ? MXP_FEW_MAX : MXP_FEWEST_MAX) * SPAN;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2 * S_BYTES;
    static constexpr int EPI_WARPS = FEW || KIND == MXP_LONG ? 4 : SPAN == 64 ? 12 : 8;
    static constexpr int STAGES = (KIND == MXP_FEWEST ? 4 : KIND == MXP_FEW ? 8 : KIND == MXP_LONG ? 10 : SPAN == 64 ? 6 : 8) / GROUPS;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int OUT_BYTES = FEW ? 0 : EPI_WARPS * MXP_OUT_BYTES;
    static constexpr int TERM_COUNT = FEW ? MXP_FEW_MAX : MXP_B, TERMS = EPI_WARPS * TERM_COUNT * 4;
    static constexpr int TMEM_COLS = 512 / CTAS, ACC_COLS = !FEW ? 384 : TMEM_COLS / 2;
    static constexpr int SF_SLOTS = (TMEM_COLS - ACC_COLS) / 8, MAX_ACCS = ACC_COLS / 16;
    static constexpr int SMEM = STAGES * STAGE_BYTES + OUT_BYTES + TERMS + 1024 /*barriers*/ + 1024 /*alignment slack*/;
    static_assert(STAGE_BYTES % 1024 == 0 && CTAS * (SMEM + 1024) <= 228 * 1024, "");
    static_assert((2 * STAGES + 2 * MAX_ACCS + 1) * 8 + 16 <= 1024, "");
};

struct MxProductArgs {
    const uint8_t* a_scales;  // of the M side
    const uint8_t* b_scales;
    const float* norms;
    const float* q_norms;
    void* out;
    int64_t ld;
    int* d_error;
    int n, nq, groups, metric;
    int b_rows, box_b;        // rows of the N side, and as many as a load brings
    unsigned units;           // tiles of 128 rows by chunks of 128 queries
    int chunks, block, acc_cols;
    bool wide;                // rows of the result begin at multiples of 16 bytes
};

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// A wait of a whole warp, with one answer.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* d_error) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, d_error));
}
// For a CTA that gives up: waits, whatever its flag says, until `fills` loads in turn into a ring of `n` have landed.
__device__ __forceinline__ void mbar_wait_landed(uint64_t* bars, uint32_t n, uint32_t fills) {
    const long long t0 = clock64();
    for (uint32_t s = 0; s < n; ++s) {
        const uint32_t of_this = fills / n + (s < fills % n);
        while (of_this && !mbar_try_wait(&bars[s], (of_this - 1) & 1u))
            if (clock64() - t0 > TC_WAIT_CYCLES) return;
    }
}
// The MMAs are issued by a whole warp, whose elected lane (the same each time) does it: what a single lane computes on its own does not get into the uniform registers that these
// instructions take their operands from without one instruction, and its latency, for each.
// Only whole warps may call these: the election waits for all 32 lanes, without a bound, so whatever leads to them has one answer for the warp (mbar_wait_warp).
// 32 rows of 16 bytes into four columns of 32 lanes, the same for each quarter of the lanes.
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xFFFFFFFF;\n\t"
        "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc)
        : "memory");
}
__device__ __forceinline__ void tc_mma_mxf4(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xFFFFFFFF;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_commit_warp(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xFFFFFFFF;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
// Descriptor of a K-major tile of SPAN-byte rows, swizzled over the span: groups of 8 rows one behind the other.
template <int SPAN>
__device__ __forceinline__ uint64_t mx_tile_desc(uint32_t saddr) {
    constexpr uint32_t hi = ((8u * SPAN) >> 4) | (1u << 14) | ((SPAN == 128 ? 2u : 4u) << 29);
    return ((uint64_t)hi << 32) | ((saddr & 0x3FFFFu) >> 4);
}
// Descriptor of a scale tile: 32 rows of 16 bytes, 8 rows every 128 bytes, no swizzle.
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t saddr) {
    constexpr uint32_t hi = (128u >> 4) | (1u << 14);
    return ((uint64_t)hi << 32) | (8ull << 16) | ((saddr & 0x3FFFFu) >> 4);
}
// e2m1 by e2m1 (type 1 each), e8m0 scales (bit 23), both K-major; the scale bytes of the first or the second half of a group (id 0 or 2).
__device__ __forceinline__ uint32_t mx_idesc(int n, uint32_t id) {
    return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(MXP_B >> 4) << 24) | (id << 29);
}

__device__ __forceinline__ void store_score(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_score(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_score(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ uint32_t pack_scores(const __half*, float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_scores(const __nv_bfloat16*, float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 1 / length; 0 for a row of zeros, whose cosines are 0; NaN where the square says too little of the length, or nothing: below 2^-126, and beyond the type.
__device__ __forceinline__ float inverse_length(float norm) {
    return norm == 0.f ? 0.f : norm >= 1.175494351e-38f && norm < INFINITY ? rsqrtf(norm) : __int_as_float(0x7FFFFFFF);
}
// What a squared norm adds to a score.
__device__ __forceinline__ float norm_term(int metric, float norm) { return metric == MX_COSINE ? inverse_length(norm) : norm; }
// Scores from dot products with one entry of one side and N of the other.
template <int N>
__device__ __forceinline__ void scores_by(int metric, uint32_t (&r)[N], float mine, const float* others) {
    if (metric == MX_COSINE) {
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * mine * others[j]);
    } else if (metric == MX_EUCLIDEAN) {
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = __float_as_uint(fmaf(2.f, __uint_as_float(r[j]), -mine) - others[j]);
    }
}

// The units, in the order in which they are taken: blocks of neighbouring tiles, a chunk of the queries after the other in each, so that the CTAs write long stretches of few queries at
// a time and a block's codes stay in L2 (1,000 x 1M float32 scores: blocks of two tiles a CTA 741 us, eight 830, all tiles at once 869, one after the other for all chunks 800).
struct MxUnit {
    int tile, chunk;
    __device__ __forceinline__ MxUnit(unsigned u, const MxProductArgs& a) {
        const unsigned b = (unsigned)(u / ((uint64_t)a.block * a.chunks)), left = (unsigned)(u - (uint64_t)b * a.block * a.chunks);
        const unsigned tiles = min((unsigned)a.block, a.units / (unsigned)a.chunks - b * (unsigned)a.block);
        chunk = (int)(left / tiles);
        tile = (int)(b * (unsigned)a.block + (left - (unsigned)chunk * tiles));
    }
};

// Rows as the M side: lanes are rows, columns queries.
template <typename Cfg, typename OUT>
__device__ __forceinline__ void mx_epilogue_few(const MxProductArgs& a, uint32_t tmem, uint64_t* acc_full, uint64_t* acc_empty, volatile int* s_abort,
                                                float* s_terms, int warp, int lane) {
    const int quarter = warp & 3;
    const uint32_t accs = Cfg::ACC_COLS / a.acc_cols;
    if (a.metric != MX_DOT) {  // of the queries; each warp for itself
        for (int q = lane; q < a.nq; q += 32) s_terms[q] = norm_term(a.metric, __ldcg(a.q_norms + q));
        __syncwarp();
    }
    bool live = true;
    uint32_t ab = 0, parity = 0;
    auto norm_of = [&](unsigned v) {
        const int64_t row = (int64_t)v * MXP_B + quarter * 32 + lane;
        return a.metric != MX_DOT && v < a.units && row < a.n ? __ldcg(a.norms + row) : 0.f;
    };
    float norm = norm_of(blockIdx.x);
    for (unsigned u = blockIdx.x; u < a.units; u += gridDim.x) {
        const int row = (int)u * MXP_B + quarter * 32 + lane;
        const float term = norm_term(a.metric, norm);
        norm = norm_of(u + gridDim.x);  // on its way while this unit is waited for
        if (live) live = mbar_wait_warp(&acc_full[ab], parity, s_abort, a.d_error);
        tc_fence_after();
        OUT* o = reinterpret_cast<OUT*>(a.out) + row;
        for (int q0 = 0; q0 < a.nq; q0 += 16) {
            uint32_t r[16];
            __syncwarp();  // rows behind the last one have not been stored
            if (live) {  // the same for the warp
                tc_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + ab * a.acc_cols + q0, r);
                tc_ld_wait();
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = 0x7FFFFFFFu;
            }
            scores_by(a.metric, r, term, s_terms + q0);
            if (row < a.n) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (q0 + j >= a.nq) break;
                    store_score(o, __uint_as_float(r[j]));
                    o += a.ld;
                }
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[ab]);
        if (++ab == accs) {
            ab = 0;
            parity ^= 1u;
        }
    }
}

// A piece from shared memory to `rows` of up to 32 queries, `left` of the scores; WIDE: rows begin at multiples of 16 bytes.
template <typename OUT, bool WIDE>
__device__ __forceinline__ void copy_piece(OUT* out, int64_t ld, const unsigned char* piece, int rows, int left, int lane) {
    constexpr int PER = 256 / sizeof(OUT), V = 16 / sizeof(OUT);
    if (WIDE && rows >= 32 && left >= PER) {  // sixteen lanes a row
        OUT* o = out + (lane >> 4) * ld + (lane & 15) * V;
        const unsigned char* const from = piece + (lane >> 4) * 256;
#pragma unroll
        for (int i0 = 0; i0 < 16; i0 += 8) {
            uint4 w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = *reinterpret_cast<const uint4*>(from + (i0 + i) * 512 + (((lane & 15) ^ ((i * 2 + (lane >> 4)) & 7)) << 4));
#pragma unroll
            for (int i = 0; i < 8; ++i, o += 2 * ld) *reinterpret_cast<uint4*>(o) = w[i];
        }
        return;
    }
#pragma unroll 4
    for (int i = 0; i < min(rows, 32); ++i) {
#pragma unroll
        for (int j = lane; j < PER; j += 32) {
            const OUT* const p = reinterpret_cast<const OUT*>(piece + i * 256 + (((j / V) ^ (i & 7)) << 4)) + j % V;
            if (j < left) out[i * ld + j] = *p;
        }
    }
}

// Queries as the M side: lanes are queries, columns rows.  Four warps take a unit, the next four the next one; a warp has 32 queries and stores 256 bytes of each
// at a time.
template <typename Cfg, typename OUT>
__device__ __forceinline__ void mx_epilogue_many(const MxProductArgs& a, uint32_t tmem, uint64_t* acc_full, uint64_t* acc_empty,
                                                 volatile int* s_abort, float* s_terms, unsigned char* piece, int warp, int lane) {
    constexpr int PER = 256 / sizeof(OUT);  // scores of a query in a piece
    constexpr uint32_t ACCS = Cfg::ACC_COLS / MXP_B, TURNS = Cfg::EPI_WARPS / 4;
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    bool live = true;
    float norm[MXP_B / 32], q_norm = 0.f;
    auto fetch = [&](unsigned u) {  // norms of a unit to come
        if (a.metric == MX_DOT || u >= a.units) return;
        const MxUnit at(u, a);
        const int q = at.chunk * MXP_B + quarter * 32 + lane;
        q_norm = q < a.nq ? __ldcg(a.q_norms + q) : 0.f;
#pragma unroll
        for (int i = 0; i < MXP_B / 32; ++i) {
            const int64_t row = (int64_t)at.tile * MXP_B + i * 32 + lane;
            norm[i] = row < a.n ? __ldcg(a.norms + row) : 0.f;
        }
    };
    uint32_t nth = group;  // unit of the CTA
    fetch(blockIdx.x + group * gridDim.x);
    for (unsigned u = blockIdx.x + group * gridDim.x; u < a.units; u += TURNS * gridDim.x, nth += TURNS) {
        const MxUnit at(u, a);
        const int q0 = at.chunk * MXP_B + quarter * 32, n0 = at.tile * MXP_B;
        const uint32_t ab = nth % ACCS;
        const float q_term = norm_term(a.metric, q_norm);
        if (a.metric != MX_DOT) {
#pragma unroll
            for (int i = 0; i < MXP_B / 32; ++i) s_terms[i * 32 + lane] = norm_term(a.metric, norm[i]);
            __syncwarp();
            fetch(u + TURNS * gridDim.x);
        }
        if (live) live = mbar_wait_warp(&acc_full[ab], (nth / ACCS) & 1u, s_abort, a.d_error);
        tc_fence_after();
        OUT* const o = reinterpret_cast<OUT*>(a.out) + (int64_t)q0 * a.ld + n0;
#pragma unroll 1
        for (int p0 = 0; p0 < MXP_B; p0 += PER) {
#pragma unroll 1
            for (int c0 = 0; c0 < PER; c0 += 32) {
                uint32_t r[32];
                if (live) {  // the same for the warp
                    tc_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + ab * MXP_B + p0 + c0, r);
                    tc_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0x7FFFFFFFu;
                }
                scores_by(a.metric, r, q_term, s_terms + p0 + c0);
                constexpr int V = 16 / sizeof(OUT);
#pragma unroll
                for (int i = 0; i < 32 / V; ++i) {  // 16 bytes each, where neither these stores nor the loads meet in a bank
                    uint4 w;
                    const uint32_t* v = r + i * V;
                    if constexpr (sizeof(OUT) == 4) {
                        w = make_uint4(v[0], v[1], v[2], v[3]);
                    } else {
                        const OUT* t = nullptr;
                        w = make_uint4(pack_scores(t, __uint_as_float(v[0]), __uint_as_float(v[1])), pack_scores(t, __uint_as_float(v[2]), __uint_as_float(v[3])),
                                       pack_scores(t, __uint_as_float(v[4]), __uint_as_float(v[5])), pack_scores(t, __uint_as_float(v[6]), __uint_as_float(v[7])));
                    }
                    *reinterpret_cast<uint4*>(piece + lane * 256 + (((c0 / V + i) ^ (lane & 7)) << 4)) = w;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (p0 + PER >= MXP_B && lane == 0) mbar_arrive(&acc_empty[ab]);
            if (a.wide) copy_piece<OUT, true>(o + p0, a.ld, piece, a.nq - q0, a.n - n0 - p0, lane);
            else copy_piece<OUT, false>(o + p0, a.ld, piece, a.nq - q0, a.n - n0 - p0, lane);
            __syncwarp();
        }
    }
}

template <int SPAN, typename OUT, MxpKind KIND>
__global__ void __launch_bounds__((MxpCfg<SPAN, KIND>::THREADS), (MxpCfg<SPAN, KIND>::CTAS))
mx_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, MxProductArgs a, KernelBefore before) {
    behind_kernel_before(before);
    using Cfg = MxpCfg<SPAN, KIND>;
    constexpr int STAGES = Cfg::STAGES;
    constexpr bool FEW = Cfg::FEW;
    extern __shared__ unsigned char mxp_smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mxp_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* s_out = base + (size_t)STAGES * Cfg::STAGE_BYTES;
    float* s_terms = reinterpret_cast<float*>(s_out + Cfg::OUT_BYTES);
    uint64_t* full = reinterpret_cast<uint64_t*>(s_out + Cfg::OUT_BYTES + Cfg::TERMS);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + Cfg::MAX_ACCS;
    uint64_t* drained = acc_empty + Cfg::MAX_ACCS;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    uint32_t* s_fills = s_tmem + 2;  // stages that have been loaded
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t accs = Cfg::ACC_COLS / a.acc_cols;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t b = 0; b < accs; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 4);
        }
        mbar_init(drained, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(Cfg::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, parity = 1, fills = 0;
            bool live = true;
            const uint32_t bytes = Cfg::A_BYTES + (uint32_t)(a.box_b * SPAN);
            for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
                const MxUnit at(u, a);
                const int ia = FEW ? at.tile : at.chunk, ib = FEW ? at.chunk : at.tile;
                for (int g = 0; g < a.groups; g += Cfg::GROUPS) {
                    if (!mbar_wait(&empty[s], parity, s_abort, a.d_error)) { live = false; break; }
                    unsigned char* st = base + (size_t)s * Cfg::STAGE_BYTES;
                    const uint32_t scales = (uint32_t)min(Cfg::GROUPS, a.groups - g) * MX_TILE_BYTES;
                    mbar_expect_tx(&full[s], bytes + 2 * scales);
                    tma_load_2d(st, &tmA, &full[s], g * 64, ia * MXP_B);
                    tma_load_2d(st + Cfg::A_BYTES, &tmB, &full[s], g * 64, ib * MXP_B);
                    bulk_load(st + Cfg::A_BYTES + Cfg::B_BYTES, a.a_scales + ((size_t)ia * a.groups + g) * MX_TILE_BYTES, scales, &full[s]);
                    bulk_load(st + Cfg::A_BYTES + Cfg::B_BYTES + Cfg::S_BYTES, a.b_scales + ((size_t)ib * a.groups + g) * MX_TILE_BYTES,
                              scales, &full[s]);
                    ++fills;
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            *s_fills = fills;
        }
    } else if (warp == 1) {
        uint32_t s = 0, parity = 0, ab = 0, acc_parity = 1, slot = 0;
        bool live = true;
        for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
            const MxUnit at(u, a);
            const int ib = FEW ? at.chunk : at.tile;
            const int n_mma = min(MXP_B, (a.b_rows - ib * MXP_B + 15) & ~15);
            if (!mbar_wait_warp(&acc_empty[ab], acc_parity, s_abort, a.d_error)) break;
            tc_fence_after();
            const uint32_t d_tmem = tmem + ab * a.acc_cols;
            const uint32_t id0 = mx_idesc(n_mma, 0), id1 = mx_idesc(n_mma, 2);
            for (int g0 = 0; g0 < a.groups; g0 += Cfg::GROUPS) {
                if (!mbar_wait_warp(&full[s], parity, s_abort, a.d_error)) { live = false; break; }
                tc_fence_after();
                const uint32_t st = smem_u32(base + (size_t)s * Cfg::STAGE_BYTES);
                const uint64_t da = mx_tile_desc<SPAN>(st), db = mx_tile_desc<SPAN>(st + Cfg::A_BYTES);
                const uint64_t dsa = mx_scale_desc(st + Cfg::A_BYTES + Cfg::B_BYTES), dsb = dsa + (Cfg::S_BYTES >> 4);
                auto group = [&](int g) {
                    const uint32_t sfa = tmem + Cfg::ACC_COLS + slot * 8, sfb = sfa + 4;
                    if (++slot == Cfg::SF_SLOTS) slot = 0;
                    tc_copy_scales(sfa, dsa + g * (MX_TILE_BYTES >> 4));
                    tc_copy_scales(sfb, dsb + g * (MX_TILE_BYTES >> 4));
                    tc_mma_mxf4(d_tmem, da + g * 4, db + g * 4, id0, sfa, sfb, (g0 | g) != 0);
                    tc_mma_mxf4(d_tmem, da + g * 4 + 2, db + g * 4 + 2, id1, sfa, sfb, 1u);
                };
                if (Cfg::GROUPS == 1 || g0 + 1 == a.groups) {
                    group(0);
                } else {
                    group(0);
                    group(1);
                }
                tc_commit_warp(&empty[s]);
                if (++s == STAGES) { s = 0; parity ^= 1u; }
            }
            if (live) tc_commit_warp(&acc_full[ab]);
            if (++ab == accs) { ab = 0; acc_parity ^= 1u; }
        }
    } else {
        float* const terms = s_terms + (warp - 2) * Cfg::TERM_COUNT;
        if constexpr (FEW) mx_epilogue_few<Cfg, OUT>(a, tmem, acc_full, acc_empty, s_abort, terms, warp, lane);
        else mx_epilogue_many<Cfg, OUT>(a, tmem, acc_full, acc_empty, s_abort, terms, s_out + (warp - 2) * MXP_OUT_BYTES, warp, lane);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*s_abort) {  // all roles are done: what they issued may not be
        if (threadIdx.x == 0) mbar_wait_landed(full, STAGES, *s_fills);
        if (warp == 1) {
            tc_commit_warp(drained);
            mbar_wait_landed(drained, 1, 1);
        }
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TMEM_COLS) : "memory");
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
inline CUtensorMap mx_codes_map(const uint8_t* codes, int rows, int groups, int span, int box_rows) {
    CUtensorMap m;
    PFN_encodeTiled enc = get_encode_tiled();
    cuuint64_t dims[2] = {(cuuint64_t)groups * 64, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)groups * 64};
    cuuint32_t box[2] = {(cuuint32_t)span, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    if (!enc || enc(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        fail(CULSH_ERR_CUDA, "no tensor map for %d rows of %d groups", rows, groups);
    return m;
}

template <int SPAN, typename OUT, MxpKind KIND>
inline void mx_product_launch(const CtxPtr& c, const uint8_t* codes, const uint8_t* q_codes, MxProductArgs a, cudaStream_t stream) {
    using Cfg = MxpCfg<SPAN, KIND>;
    constexpr bool FEW = Cfg::FEW;
    const CUtensorMap tx = mx_codes_map(codes, a.n, a.groups, SPAN, FEW ? MXP_B : a.box_b);
    const CUtensorMap tq = mx_codes_map(q_codes, a.nq, a.groups, SPAN, FEW ? a.box_b : MXP_B);
    auto kern = mx_product_kernel<SPAN, OUT, KIND>;
    static thread_local uint64_t ready = 0;  // devices whose limit is set
    if (c->device >= 64 || !(ready >> c->device & 1)) {
        CU_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        if (c->device < 64) ready |= 1ull << c->device;
    }
    launch_next(stream, mx_product_kernel<SPAN, OUT, KIND>, std::min<unsigned>(a.units, (unsigned)(c->sm_count * Cfg::CTAS)), (unsigned)Cfg::THREADS,
                (size_t)Cfg::SMEM, FEW ? tx : tq, FEW ? tq : tx, a);
    KERNEL_CHECK();
}

template <typename OUT>
inline void mx_product(const CtxPtr& c, const uint8_t* q_codes, const uint8_t* q_scales, const float* q_norms, int nq, const uint8_t* codes,
                       const uint8_t* scales, const float* norms, int n, int d, int metric, OUT* out, int64_t ld, int* d_error, cudaStream_t stream) {
    const bool few = nq <= MXP_FEW_MAX;
    MxProductArgs a{};
    a.a_scales = few ? scales : q_scales, a.b_scales = few ? q_scales : scales;
    a.norms = norms, a.q_norms = q_norms, a.out = out, a.ld = ld, a.d_error = d_error;
    a.n = n, a.nq = nq, a.groups = mx_groups(d), a.metric = metric;
    a.b_rows = few ? nq : n;
    a.box_b = (int)std::min<int64_t>(MXP_B, ((int64_t)a.b_rows + 15) & ~15);
    a.chunks = (int)ceil_div(nq, MXP_B);
    if ((uint64_t)mx_tiles(n) * a.chunks >= (1ull << 31)) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", nq, n);
    a.units = mx_tiles(n) * (unsigned)a.chunks;
    a.block = 2 * c->sm_count;
    a.acc_cols = !few ? MXP_B : nq <= 16 ? 16 : nq <= 32 ? 32 : 64;
    a.wide = aligned16(out, ld * (int64_t)sizeof(OUT));
    auto go = [&](auto kind) {
        constexpr MxpKind K = decltype(kind)::value;
        if constexpr (K == MXP_LONG) {
            mx_product_launch<128, OUT, K>(c, codes, q_codes, a, stream);
        } else {
            if (a.groups > 1) mx_product_launch<128, OUT, K>(c, codes, q_codes, a, stream);
            else mx_product_launch<64, OUT, K>(c, codes, q_codes, a, stream);
        }
    };
    if (nq <= MXP_FEWEST_MAX) go(std::integral_constant<MxpKind, MXP_FEWEST>());
    else if (few) go(std::integral_constant<MxpKind, MXP_FEW>());
    else if (a.groups >= MXP_LONG_GROUPS) go(std::integral_constant<MxpKind, MXP_LONG>());
    else go(std::integral_constant<MxpKind, MXP_MANY>());
}

}  // namespace culsh_b200
