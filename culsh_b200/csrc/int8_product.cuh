// Scores of queries against all rows, both in 8-bit integers (int8_rows.cuh), and against lists of candidates.
//
//   A = sum_k cq_k cx_k, exact in int32;   dot = A sq sx,   cosine = A / (sqrt(squares_q) sqrt(squares_x)),   euclidean = 2 A sq sx - sq^2 squares_q - sx^2 squares_x
#pragma once

#include "int8_rows.cuh"
#include "tc_gemm.cuh"

namespace culsh_b200 {

// What a row's scale and squares put into a score: a factor of A, and a term that is taken off.
__device__ __forceinline__ float2 i8_terms(int metric, float scale, int squares) {
    if (metric == MX_COSINE) return make_float2(squares > 0 ? __frsqrt_rn((float)squares) : squares == 0 ? 0.f : __int_as_float(0x7FFFFFFF), 0.f);
    return make_float2(scale, metric == MX_EUCLIDEAN ? (float)squares * (scale * scale) : 0.f);
}
__device__ __forceinline__ float i8_score(int metric, int dot, float2 q, float2 x) {
    const float v = (float)dot * (q.x * x.x);
    return metric == MX_EUCLIDEAN ? fmaf(2.f, v, -q.y) - x.y : v;
}

struct I8ProductArgs {
    int* d_error;
    unsigned units;
    uint32_t idesc;
    int n, nq, kb, metric, chunks, block;
    unsigned tiles;
    const float *scales, *q_scales;
    const int32_t *squares, *q_squares;
    void* out;
    int64_t ld;
    bool wide;
};
constexpr int I8_BN = 256;
struct I8Unit {
    static constexpr int tiles = 1, k0 = 0;
    int tile, chunk, k1;
    __device__ __forceinline__ I8Unit(const I8ProductArgs& a, unsigned u) {  // blocks of neighbouring tiles, a chunk of the queries after the other in each
        const unsigned b = (unsigned)(u / ((uint64_t)a.block * a.chunks)), left = (unsigned)(u - (uint64_t)b * a.block * a.chunks);
        const unsigned here = min((unsigned)a.block, a.tiles - b * (unsigned)a.block);
        chunk = (int)(left / here);
        tile = (int)(b * (unsigned)a.block + (left - (unsigned)chunk * here));
        k1 = a.kb;
    }
};
template <typename OUT, bool PAIRS>
struct I8ProductPolicy {
    static constexpr bool A_MN = false, B_MN = false, I8 = true, PARTS = true, PAIR = PAIRS;
    static constexpr int BN = I8_BN, PART = BN / 2, SEGMENT = 0, EPI_WARPS = 8, EPI_BYTES = EPI_WARPS * (MXP_OUT_BYTES + PART * 8);
    using Pairs = PlanePairs<1>;
    using Args = I8ProductArgs;
    using Unit = I8Unit;
    static __device__ __forceinline__ void load(const Args&, const Unit& u, int, int, int, int k, const CUtensorMap* ta, const CUtensorMap* tb, unsigned char* sa, unsigned char* sb,
                                                uint32_t bar, int rank) {
        tma_load_3d<PAIR>(sa, ta, bar, k * 128, u.chunk * (PAIR ? 2 * TG_M : TG_M) + rank * TG_M, 0);
        tma_load_3d<PAIR>(sb, tb, bar, k * 128, u.tile * BN + rank * (BN / 2), 0);
    }
    static __device__ __forceinline__ int n_mma(const Args& a, const Unit& u, int) { return min(BN, (a.n - u.tile * BN + 15) & ~15); }
    struct Epilogue {
        int quarter, group, lane, rank;
        unsigned char* piece;
        float2* terms;
        __device__ __forceinline__ Epilogue(const Args&, unsigned char* smem, int warp, int quarter_, int group_, int lane_, int rank_)
            : quarter(quarter_), group(group_), lane(lane_), rank(rank_), piece(smem + warp * MXP_OUT_BYTES),
              terms(reinterpret_cast<float2*>(smem + EPI_WARPS * MXP_OUT_BYTES) + warp * PART) {}
        __device__ __forceinline__ void unit_begin(const Args&, const Unit&) {}
        __device__ __forceinline__ void unit_end(const Args&, const Unit&) {}
        template <typename D>
        __device__ __forceinline__ void tile(const Args& a, const Unit& u, int, uint32_t taddr, bool live, bool, D&& done) {
            constexpr int PER = 256 / sizeof(OUT), V = 16 / sizeof(OUT);  // scores of a query in a piece, in a store
            const int q0 = u.chunk * (PAIR ? 2 * TG_M : TG_M) + rank * TG_M + quarter * 32, n0 = u.tile * BN + group * PART;
            if (q0 >= a.nq || n0 >= a.n) {
                done();
                return;
            }
            const int q = q0 + lane;
            float2 mine = q < a.nq ? i8_terms(a.metric, __ldcg(a.q_scales + q), __ldcg(a.q_squares + q)) : make_float2(0.f, 0.f);
            if (!live) mine.x = __int_as_float(0x7FFFFFFF);
#pragma unroll
            for (int i = lane; i < PART; i += 32) terms[i] = n0 + i < a.n ? i8_terms(a.metric, __ldcg(a.scales + n0 + i), __ldcg(a.squares + n0 + i)) : make_float2(0.f, 0.f);
            __syncwarp();
            OUT* const o = reinterpret_cast<OUT*>(a.out) + (int64_t)q0 * a.ld + n0;
#pragma unroll 1
            for (int p0 = 0; p0 < PART; p0 += PER) {
#pragma unroll 1
                for (int c0 = 0; c0 < PER; c0 += 32) {
                    uint32_t r[32];
                    tg_read(taddr + p0 + c0, live, r);
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(i8_score(a.metric, (int)r[j], mine, terms[p0 + c0 + j]));
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
                if (p0 + PER >= PART) done();
                __syncwarp();
                if (a.wide) copy_piece<OUT, true>(o + p0, a.ld, piece, a.nq - q0, a.n - n0 - p0, lane);
                else copy_piece<OUT, false>(o + p0, a.ld, piece, a.nq - q0, a.n - n0 - p0, lane);
                __syncwarp();
            }
        }
    };
};

struct I8ScoreArgs {
    const int8_t *codes, *q_codes;
    const float *scales, *q_scales;
    const int32_t *squares, *q_squares;
    const int32_t* ids;
    const int64_t* offsets;
    float* out;
    int64_t total;
    int n, nq, pitch, metric, lanes;
};
// The list that entry c belongs to, from list `low` on: the last one that begins at or before it.
__device__ __forceinline__ int i8_owner(const int64_t* offsets, int low, int nq, int64_t c) {
    int high = nq;
    while (high - low > 1) {
        const int mid = low + (high - low) / 2;
        if (__ldcg(offsets + mid) <= c) low = mid;
        else high = mid;
    }
    return low;
}
// A warp takes 32 candidates after the others; `lanes` threads (a power of two up to 32) one of them, 16 bytes of its row each at a time.
__global__ void __launch_bounds__(256) i8_score_kernel(I8ScoreArgs a, KernelBefore before) {
    behind_kernel_before(before);
    const int lane = threadIdx.x & 31, at = lane & (a.lanes - 1), groups = 32 / a.lanes, group = lane / a.lanes;
    const int64_t warps = (int64_t)gridDim.x * 8, spans = (a.total + 31) / 32;
    for (int64_t s = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); s < spans; s += warps) {
        const int64_t c = s * 32 + lane;
        const bool in = c < a.total;
        const int id = in ? __ldcg(a.ids + c) : -1;
        const int owner = i8_owner(a.offsets, 0, a.nq, in ? c : a.total - 1);
        float score = __int_as_float(0x7FFFFFFF);
        for (int i = 0; i < a.lanes; ++i) {
            const int which = i * groups + group;
            const int row = __shfl_sync(0xFFFFFFFFu, id, which), q = __shfl_sync(0xFFFFFFFFu, owner, which);
            int dot = 0;
            if ((unsigned)row < (unsigned)a.n) {
                const uint4* const x = reinterpret_cast<const uint4*>(a.codes + (int64_t)row * a.pitch);
                const uint4* const y = reinterpret_cast<const uint4*>(a.q_codes + (int64_t)q * a.pitch);
                for (int k = at; k < a.pitch / 16; k += a.lanes) {
                    const uint4 v = __ldcg(x + k), w = __ldcg(y + k);
                    dot = __dp4a((int)v.x, (int)w.x, dot);
                    dot = __dp4a((int)v.y, (int)w.y, dot);
                    dot = __dp4a((int)v.z, (int)w.z, dot);
                    dot = __dp4a((int)v.w, (int)w.w, dot);
                }
            }
            for (int o = 1; o < a.lanes; o *= 2) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
            const int mine = __shfl_sync(0xFFFFFFFFu, dot, (lane % groups) * a.lanes);
            if (lane / groups == i && (unsigned)id < (unsigned)a.n)
                score = i8_score(a.metric, mine, i8_terms(a.metric, __ldcg(a.q_scales + owner), __ldcg(a.q_squares + owner)),
                                 i8_terms(a.metric, __ldcg(a.scales + id), __ldcg(a.squares + id)));
        }
        if (in) a.out[c] = score;
    }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
template <typename OUT>
inline void i8_product(const CtxPtr& c, const int8_t* q_codes, const float* q_scales, const int32_t* q_squares, int nq, const int8_t* codes, const float* scales,
                       const int32_t* squares, int n, int d, int metric, OUT* out, int64_t ld, int* d_error, cudaStream_t stream) {
    I8ProductArgs a{};
    a.d_error = d_error, a.idesc = tg_idesc(TG_I8, false, false);
    a.n = n, a.nq = nq, a.kb = (int)ceil_div(i8_pitch(d), 128), a.metric = metric;
    const bool pairs = nq > TG_M;
    a.chunks = (int)ceil_div(nq, pairs ? 2 * TG_M : TG_M), a.tiles = (unsigned)ceil_div(n, I8_BN), a.block = 2 * c->sm_count;
    if ((uint64_t)a.tiles * a.chunks >= (1ull << 31)) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", nq, n);
    a.units = a.tiles * (unsigned)a.chunks;
    a.scales = scales, a.q_scales = q_scales, a.squares = squares, a.q_squares = q_squares, a.out = out, a.ld = ld;
    a.wide = aligned16(out, ld * (int64_t)sizeof(OUT));
    const int pitch = i8_pitch(d);
    const CUtensorMap tq = tg_map(q_codes, TG_I8, nq, pitch, pitch, 1, 0, TG_M), tx = tg_map(codes, TG_I8, n, pitch, pitch, 1, 0, pairs ? I8_BN / 2 : I8_BN);
    if (pairs) tc_gemm<I8ProductPolicy<OUT, true>>(c, tq, tx, a, stream);
    else tc_gemm<I8ProductPolicy<OUT, false>>(c, tq, tx, a, stream);
}

inline void i8_score_lists(const CtxPtr& c, I8ScoreArgs a, cudaStream_t stream) {
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes * 16 < a.pitch) a.lanes *= 2;
    const size_t grid = std::min<size_t>(ceil_div(a.total, 256), (size_t)c->sm_count * 8 * 8);
    launch_next(stream, i8_score_kernel, grid, 256u, 0, a);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
