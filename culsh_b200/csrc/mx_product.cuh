// Scores of queries against all rows, both in microscaled 4-bit floating point (mx_rows.cuh): out[q][row] = sum_k q^_k x^_k, or the cosine, or the
// negative squared distance, on the 5th-generation tensor cores (tcgen05.mma kind::mxf4 with block scales, fp32 accumulators in tensor memory).
//
// The rows are the M side (a tile of 128), the queries the N side (chunks of up to 128): an accumulator lane is a row, so a warp's stores of a query are 32
// neighbouring scores.  Codes come by TMA, swizzled; scale tiles of 512 bytes (128 rows by 4 blocks) lie in memory as the tensor cores
// take them and go from shared into tensor memory by tcgen05.cp, issued by the thread that issues the MMAs, in front of the two MMAs (64 values each) that read them.
//
// One persistent CTA per SM, 10 warps: TMA producer, MMA issuer, eight of epilogue; three accumulators of 128 columns in turn.  Every wait is bounded
// (mbar_wait); a CTA whose wait ran out records it and fills what it has not done with NaN.  No load uses cluster multicast.
#pragma once

#include <algorithm>

#include "mx_rows.cuh"
#include "tc_ptx.cuh"

namespace culsh_b200 {

enum MxMetric : int { MX_DOT = 0, MX_COSINE = 1, MX_EUCLIDEAN = 2 };

constexpr int MXP_BM = 128, MXP_BN = 128, MXP_ACCS = 3, MXP_EPI_WARPS = 8, MXP_THREADS = 64 + 32 * MXP_EPI_WARPS;
constexpr int MXP_SF_COL = MXP_ACCS * MXP_BN, MXP_SF_SLOTS = (512 - MXP_SF_COL) / 8;

// SPAN: bytes of a row in a stage, the swizzle span: 64 (one group) or 128 (two).
template <int SPAN>
struct MxpCfg {
    static constexpr int GROUPS = SPAN / 64;
    static constexpr int A_BYTES = MXP_BM * SPAN, B_BYTES = MXP_BN * SPAN, S_BYTES = GROUPS * MX_TILE_BYTES;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2 * S_BYTES;
    static constexpr int STAGES = SPAN == 128 ? 6 : 12;
    static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*barriers*/ + 1024 /*alignment slack*/;
    static_assert(STAGE_BYTES % 1024 == 0, "");
    static_assert((2 * STAGES + 2 * MXP_ACCS) * 8 + 16 <= 1024, "");
};

struct MxProductArgs {
    const uint8_t* scales;
    const uint8_t* q_scales;
    const float* norms;
    const float* q_norms;
    void* out;
    int64_t ld;
    int* d_error;
    int n, nq, groups, metric, box_q;
    unsigned units;
    int chunks;
    bool pairs;  // two scores of 16 bits can be stored at once
};

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// 32 rows of 16 bytes into four columns of 32 lanes, the same for each quarter of the lanes.
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void tc_mma_mxf4(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
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
    return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(MXP_BM >> 4) << 24) | (id << 29);
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

// 1 / length; 0 for a row of zeros, whose cosines are 0.
__device__ __forceinline__ float inverse_length(float norm) { return norm == 0.f ? 0.f : 1.f / sqrtf(norm); }

template <int SPAN, typename OUT>
__global__ void __launch_bounds__(MXP_THREADS, 1)
mx_product_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmQ, MxProductArgs a) {
    using Cfg = MxpCfg<SPAN>;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ unsigned char mxp_smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mxp_smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(base + (size_t)STAGES * Cfg::STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + MXP_ACCS;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(acc_empty + MXP_ACCS);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < MXP_ACCS; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], MXP_EPI_WARPS);
        }
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
    const uint32_t tmem = *s_tmem;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, parity = 1;
            bool live = true;
            const uint32_t q_bytes = (uint32_t)(a.box_q * SPAN);
            for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
                const int tile = (int)(u / (unsigned)a.chunks), c = (int)(u - (unsigned)tile * (unsigned)a.chunks);
                for (int g = 0; g < a.groups; g += Cfg::GROUPS) {
                    if (!mbar_wait(&empty[s], parity, s_abort, a.d_error)) { live = false; break; }
                    unsigned char* st = base + (size_t)s * Cfg::STAGE_BYTES;
                    mbar_expect_tx(&full[s], Cfg::A_BYTES + q_bytes + 2 * Cfg::S_BYTES);
                    tma_load_2d(st, &tmX, &full[s], g * 64, tile * MXP_BM);
                    tma_load_2d(st + Cfg::A_BYTES, &tmQ, &full[s], g * 64, c * MXP_BN);
                    bulk_load(st + Cfg::A_BYTES + Cfg::B_BYTES, a.scales + ((size_t)tile * a.groups + g) * MX_TILE_BYTES, Cfg::S_BYTES, &full[s]);
                    bulk_load(st + Cfg::A_BYTES + Cfg::B_BYTES + Cfg::S_BYTES, a.q_scales + ((size_t)c * a.groups + g) * MX_TILE_BYTES,
                              Cfg::S_BYTES, &full[s]);
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t s = 0, parity = 0, ab = 0, acc_parity = 1, slot = 0;
            bool live = true;
            for (unsigned u = blockIdx.x; u < a.units && live; u += gridDim.x) {
                const int c = (int)(u % (unsigned)a.chunks);
                const int n_mma = min(MXP_BN, (a.nq - c * MXP_BN + 15) & ~15);
                if (!mbar_wait(&acc_empty[ab], acc_parity, s_abort, a.d_error)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem + ab * MXP_BN;
                const uint32_t id0 = mx_idesc(n_mma, 0), id1 = mx_idesc(n_mma, 2);
                for (int g0 = 0; g0 < a.groups; g0 += Cfg::GROUPS) {
                    if (!mbar_wait(&full[s], parity, s_abort, a.d_error)) { live = false; break; }
                    tc_fence_after();
                    const uint32_t st = smem_u32(base + (size_t)s * Cfg::STAGE_BYTES);
                    const uint64_t da = mx_tile_desc<SPAN>(st), db = mx_tile_desc<SPAN>(st + Cfg::A_BYTES);
                    const uint64_t dsa = mx_scale_desc(st + Cfg::A_BYTES + Cfg::B_BYTES), dsb = dsa + (Cfg::S_BYTES >> 4);
#pragma unroll
                    for (int g = 0; g < Cfg::GROUPS; ++g) {
                        const uint32_t sfa = tmem + MXP_SF_COL + slot * 8, sfb = sfa + 4;
                        if (++slot == MXP_SF_SLOTS) slot = 0;
                        tc_copy_scales(sfa, dsa + g * (MX_TILE_BYTES >> 4));
                        tc_copy_scales(sfb, dsb + g * (MX_TILE_BYTES >> 4));
                        tc_mma_mxf4(d_tmem, da + g * 4, db + g * 4, id0, sfa, sfb, (g0 | g) != 0);
                        tc_mma_mxf4(d_tmem, da + g * 4 + 2, db + g * 4 + 2, id1, sfa, sfb, 1u);
                    }
                    tc_commit(&empty[s]);
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
                if (live) tc_commit(&acc_full[ab]);
                if (++ab == MXP_ACCS) { ab = 0; acc_parity ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t ab = 0, acc_parity = 0;
        bool live = true;
        OUT* const out = reinterpret_cast<OUT*>(a.out);
        for (unsigned u = blockIdx.x; u < a.units; u += gridDim.x) {
            const int tile = (int)(u / (unsigned)a.chunks), c = (int)(u - (unsigned)tile * (unsigned)a.chunks);
            const int row = tile * MXP_BM + quarter * 32 + lane;
            const bool row_ok = row < a.n;
            const float norm = a.metric != MX_DOT && row_ok ? __ldg(a.norms + row) : 0.f;
            const float x_term = a.metric == MX_COSINE ? inverse_length(norm) : norm;
            const int q_here = min(MXP_BN, a.nq - c * MXP_BN), blocks = (q_here + 15) >> 4, split = (blocks + 1) >> 1;
            if (live) live = mbar_wait(&acc_full[ab], acc_parity, s_abort, a.d_error);
            tc_fence_after();
            for (int b = half ? split : 0; b < (half ? blocks : split); ++b) {
                uint32_t r[16];
                if (live) {  // the same for the warp
                    tc_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + ab * MXP_BN + b * 16, r);
                    tc_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[j] = 0x7FFFFFFFu;
                }
                const int q0 = c * MXP_BN + b * 16;
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    v[j] = __uint_as_float(r[j]);
                    if (a.metric != MX_DOT) {
                        const float qn = __ldg(a.q_norms + min(q0 + j, a.nq - 1));
                        v[j] = a.metric == MX_COSINE ? v[j] * x_term * inverse_length(qn) : 2.f * v[j] - qn - x_term;
                    }
                }
                OUT* o = out + (int64_t)q0 * a.ld + row;
                if constexpr (sizeof(OUT) == 2) {
                    if (a.pairs) {
                        const bool odd = lane & 1;
                        o -= odd;
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[j] : v[j + 1], 1);
                            const float lo = odd ? other : v[j], hi = odd ? v[j + 1] : other;
                            if (q0 + j + odd < a.nq) {
                                OUT* p = o + (int64_t)(j + odd) * a.ld;
                                if ((row | 1) < a.n) *reinterpret_cast<uint32_t*>(p) = pack_scores(p, lo, hi);
                                else if ((row & ~1) < a.n) store_score(p, lo);
                            }
                        }
                        continue;
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (row_ok && q0 + j < a.nq) store_score(o + (int64_t)j * a.ld, v[j]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[ab]);
            if (++ab == MXP_ACCS) { ab = 0; acc_parity ^= 1u; }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
inline CUtensorMap mx_codes_map(const uint8_t* codes, int n, int groups, int span, int box_rows) {
    CUtensorMap m;
    PFN_encodeTiled enc = get_encode_tiled();
    cuuint64_t dims[2] = {(cuuint64_t)groups * 64, (cuuint64_t)n};
    cuuint64_t strides[1] = {(cuuint64_t)groups * 64};
    cuuint32_t box[2] = {(cuuint32_t)span, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    if (!enc || enc(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        fail(CULSH_ERR_CUDA, "no tensor map for %d rows of %d groups", n, groups);
    return m;
}

template <int SPAN, typename OUT>
inline void mx_product_launch(const CtxPtr& c, const uint8_t* codes, const uint8_t* q_codes, MxProductArgs a, cudaStream_t stream) {
    using Cfg = MxpCfg<SPAN>;
    const CUtensorMap tx = mx_codes_map(codes, a.n, a.groups, SPAN, MXP_BM), tq = mx_codes_map(q_codes, a.nq, a.groups, SPAN, a.box_q);
    auto kern = mx_product_kernel<SPAN, OUT>;
    static thread_local uint64_t ready = 0;  // devices whose limit is set
    if (c->device >= 64 || !(ready >> c->device & 1)) {
        CU_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        if (c->device < 64) ready |= 1ull << c->device;
    }
    kern<<<std::min<unsigned>(a.units, (unsigned)c->sm_count), MXP_THREADS, Cfg::SMEM, stream>>>(tx, tq, a);
    KERNEL_CHECK();
}

template <typename OUT>
inline void mx_product(const CtxPtr& c, const uint8_t* q_codes, const uint8_t* q_scales, const float* q_norms, int nq, const uint8_t* codes,
                       const uint8_t* scales, const float* norms, int n, int d, int metric, OUT* out, int64_t ld, int* d_error, cudaStream_t stream) {
    MxProductArgs a{};
    a.scales = scales, a.q_scales = q_scales, a.norms = norms, a.q_norms = q_norms, a.out = out, a.ld = ld, a.d_error = d_error;
    a.n = n, a.nq = nq, a.groups = mx_groups(d), a.metric = metric;
    a.box_q = std::min(MXP_BN, (nq + 15) & ~15);
    a.chunks = (int)ceil_div(nq, MXP_BN);
    if ((uint64_t)mx_tiles(n) * a.chunks >= (1ull << 31)) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", nq, n);
    a.units = mx_tiles(n) * (unsigned)a.chunks;
    a.pairs = sizeof(OUT) == 2 && (ld & 1) == 0 && ((uintptr_t)out & 3) == 0;
    if (a.groups % 2 == 0) mx_product_launch<128, OUT>(c, codes, q_codes, a, stream);
    else mx_product_launch<64, OUT>(c, codes, q_codes, a, stream);
}

}  // namespace culsh_b200
