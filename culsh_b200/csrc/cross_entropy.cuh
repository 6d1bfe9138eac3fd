// Softmax cross entropy of queries over every row, whose scores are not kept, and its gradient.
//
//   z_ij = q_i . x_j / T + b_j      lse_i = log sum_j exp(z_ij)      loss_i = lse_i - z_i,t(i)
//   G_ij = (g_i + e_i) p_ij - g_i [j = t(i)],  p = exp(z - lse)      dQ = G X / T      dX = G^T Q / T
//
// with g and e the gradients that come from the losses and from lse.  Everything is taken in powers of two: c = log2(e) / T and b log2(e).
//
// Forward: products on the tensor cores (tc_gemm.cuh), queries on the M side, so that a thread holds neighbouring scores of one query and keeps the running maximum and sum of
// a block of rows by itself; blocks are joined in 64 bits.  lse comes as two floats, of which the second is what the first leaves: a score of a thousand would leave p an error of 2^-14 otherwise.
//
// Backward: rows in pieces whose G fits L2 (four times as much in 32 bits, where six products read it); for each, G once more from the products, and two products with it.  Rows of up to 256 values of 16 bits
// keep it on the SM (ce_fused.cuh).  The target's own entry stays out of G: where p is near 1 it is a small
// difference, and where it is not, it outweighs the rest and so would its rounding to 16 bits; its coefficient g expm1(-loss) + e exp(-loss) is taken in 32 bits, and times the row or the
// query added to the sums (ce_prepare_kernel, ce_finish_kernel).  Sums of one row's gradient over its queries are taken in ascending order: nothing depends on the order of atomics.
//
// 32-bit floats are held as three bfloat16 planes each (24 bits), products as six of 16 bits; G of 32-bit inputs likewise.  G of 16-bit inputs is rounded to their type, an operand of the tensor cores: its
// errors average out over a long sum, and the result's own rounding is some eighty times as much (4,096 x 100,000 x 128: rms 2.3e-5 of 1.7e-3 in bfloat16, 2.9e-6 of 2.1e-4 in float16), where a second
// plane would double both products.  Where a few entries make the sum, both roundings are alike (1.4 times the result's).  G of half precision is scaled by a power of two that brings the
// largest coefficient to 2^15, so that p down to 2^-39 of it is there.
#pragma once

#include <cmath>
#include <type_traits>

#include "ce_fused.cuh"
#include "tc_gemm.cuh"

namespace culsh_b200 {

constexpr int CE_BN = 256, CE_PART = CE_BN / 4;  // columns of a tile, and of it for a warp
// Steps of 64 in a segment of K (tc_gemm.cuh), of the losses' scores and of the gradient's, so that p are a softmax of the same numbers: in one sum over 65,536 values the gradient's scores of 40 would
// be 3e-4 of themselves smaller, and all p 1.3e-2.  A segment's 32 adds cut off 1e-6 of a score (32 x 2^-25 of it on average, as its sum grows).  4,099 x 32,771 x 2,048 float16: losses 380 us, by
// segments of 256 values 414; gradient 1.51 ms, in one sum 1.46.  Calls of few tiles, which leave most SMs idle, have time for shorter ones: losses of 64 x 4,891 x 1,321 bfloat16 4.3e-7 off in place
// of 1.6e-6 in the same 35 us (128 x 9,000 x 4,096 33 us in place of 26).  So have those of up to 32 queries, where the rows' reads take the time and one warp in four has lanes to read: 4 x 100,000 x
// 1,024 bfloat16 1.6e-7 off in place of 8.6e-7, 53 us either way (of 64 by 768 44 in place of 41, of 128 by 200,000 x 256 39 in place of 32).
constexpr int CE_SEGMENT = 8, CE_SEGMENT_SMALL = 2;

struct CeScoreArgs {
    int* d_error;
    unsigned units;
    uint32_t idesc;
    int m, kb, segment;       // queries; steps of K, and of a segment of it
    int n0, n1;               // rows of this call
    int block, tiles_q, m_tile;  // tiles of rows in a unit; tiles of queries, and their size
    unsigned tiles_n;
    float c;
    const float* bias;        // of the rows, in powers of two, or NULL
    const int64_t* targets;   // (forward) of the queries, or -1
    // forward
    float down;               // what scores are multiplied by before differences are taken (c is as much larger)
    float2* partial;          // [m][slots]: reference and sum
    int slots;
    float* target_scores;     // [m]
    // gradient
    const float* terms;       // [m] what goes to the exponent: -lse, plus `shift`
    const float* factors;     // [m] what p is multiplied by
    int shift;
    const uint32_t* amax;     // largest magnitude among the factors, as bits (half precision only)
    const int* target_cols;   // [m] or -1
    void* G;                  // [planes][m][pitch]
    int64_t pitch, plane;
};

struct CeUnit {
    int m0, tile0, tiles, k0, k1, block;
    __device__ __forceinline__ CeUnit(const CeScoreArgs& a, unsigned u) {
        block = (int)(u / (unsigned)a.tiles_q);
        m0 = (int)(u - (unsigned)block * a.tiles_q) * a.m_tile;
        tile0 = block * a.block;
        tiles = min(a.block, (int)a.tiles_n - tile0);
        k0 = 0, k1 = a.kb;
    }
};

// Tiles of 256 rows, of a CTA or of a pair of them, and of 64 where those would leave most SMs idle.
enum CeTile : int { CE_ONE = 0, CE_PAIR = 1, CE_SMALL = 2 };
template <int PLANES, bool K_SEGMENTS, int TILE>
struct CeScoreBase {
    static constexpr bool A_MN = false, B_MN = false, I8 = false, PARTS = true, PAIR = TILE == CE_PAIR;
    static constexpr int BN = TILE == CE_SMALL ? CE_PART : CE_BN, SEGMENTS = K_SEGMENTS, EPI_WARPS = BN / 16;
    static constexpr int EPI_BYTES = EPI_WARPS * CE_PART * 4;
    using Pairs = PlanePairs<PLANES>;
    using Args = CeScoreArgs;
    using Unit = CeUnit;
    static __device__ __forceinline__ void load(const Args& a, const Unit& u, int t, int pa, int pb, int k, const CUtensorMap* ta, const CUtensorMap* tb, unsigned char* sa,
                                                unsigned char* sb, uint32_t bar, int rank) {
        tma_load_3d<PAIR>(sa, ta, bar, k * 64, u.m0 + rank * TG_M, pa);
        tma_load_3d<PAIR>(sb, tb, bar, k * 64, a.n0 + (u.tile0 + t) * BN + rank * (BN / 2), pb);
    }
    static __device__ __forceinline__ int n_mma(const Args& a, const Unit& u, int t) { return min(BN, (a.n1 - a.n0 - (u.tile0 + t) * BN + 15) & ~15); }
};

// The rows' terms of a warp's part of a tile.
__device__ __forceinline__ void ce_bias_tile(const float* bias, int n0, int n1, float* s, int lane) {
    __syncwarp();
#pragma unroll
    for (int i = lane; i < CE_PART; i += 32) s[i] = n0 + i < n1 ? __ldcg(bias + n0 + i) : -INFINITY;
    __syncwarp();
}

// The sums of a tile's segments, for a thread's columns of one lane.  WIDE: all of them at a time (few warps, which have the registers).
template <bool SEGMENTS, bool WIDE>
struct CeSums {
    static_assert(CE_PART == 64, "");
    float v[SEGMENTS ? CE_PART : 1];
    __device__ __forceinline__ void segment(const CeScoreArgs&, bool first, uint32_t taddr, bool) {
        if constexpr (SEGMENTS) {
            auto each = [&](auto&& f) {
                if constexpr (WIDE) {
                    uint32_t r[2][32];
                    tg_ld64(taddr, r);
                    tc_ld_wait();
#pragma unroll
                    for (int j = 0; j < CE_PART; ++j) f(v[j], __uint_as_float(r[j / 32][j % 32]));
                } else {
#pragma unroll
                    for (int c0 = 0; c0 < CE_PART; c0 += 16) {
                        uint32_t r[16];
                        tg_ld16(taddr + c0, r);
                        tc_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) f(v[c0 + j], __uint_as_float(r[j]));
                    }
                }
            };
            if (first) each([](float& to, float from) { to = from; });
            else each([](float& to, float from) { to += from; });
        }
    }
    // All of them, where this is the last segment: f(columns).
    template <typename F>
    __device__ __forceinline__ void read(const CeScoreArgs& a, uint32_t taddr, bool live, bool more, F&& f) {
        if constexpr (SEGMENTS) {
            CeSums::segment(a, !more, taddr, live);
            f(v);
        } else {
            uint32_t r[2][32];
            tg_ld64(taddr, r);
            tc_ld_wait();
            float x[CE_PART];
#pragma unroll
            for (int j = 0; j < CE_PART; ++j) x[j] = __uint_as_float(r[j / 32][j % 32]);
            f(x);
        }
    }
};

// A thread keeps the largest of its part of a query's scores (of the exponents, where there is a bias) and the sum of exponentials by it; the largest one's is exactly 1, and so the loss of a query
// that has but one row is exactly 0.  Of a batch, bound by the exponentials, 16 a cycle and SM: 4,096 x
// 1M x 128 bfloat16 1.34 ms, their unit busy for 77 %, the tensor pipe for 38.  (Eight warps in place of sixteen 2.0 ms; an arrival that releases to the cluster, for each tile of each warp, 1.9.)
template <int PLANES, bool BIAS, bool SEGMENTS, int TILE>
struct CeLossPolicy : CeScoreBase<PLANES, SEGMENTS, TILE> {
    static constexpr int BN = CeScoreBase<PLANES, SEGMENTS, TILE>::BN;
    struct Epilogue : CeSums<SEGMENTS, TILE == CE_SMALL> {
        int q, quarter, group, lane, rank, target;
        bool idle;
        float ref, sum;
        float* s_bias;
        __device__ __forceinline__ Epilogue(const CeScoreArgs&, unsigned char* smem, int warp, int quarter_, int group_, int lane_, int rank_)
            : quarter(quarter_), group(group_), lane(lane_), rank(rank_), s_bias(reinterpret_cast<float*>(smem) + warp * CE_PART) {}
        __device__ __forceinline__ void unit_begin(const CeScoreArgs& a, const CeUnit& u) {
            q = u.m0 + rank * TG_M + quarter * 32 + lane;
            idle = q - lane >= a.m;
            ref = -INFINITY, sum = 0.f;
            const int64_t t = q < a.m && a.targets ? __ldcg(a.targets + q) : -1;
            target = t < 0 || t >= a.n1 ? -1 : (int)t;
        }
        // x: scores, or exponents where there is a bias
        __device__ __forceinline__ void add(const CeScoreArgs& a, float (&x)[CE_PART]) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < CE_PART; j += 2) top = fmaxf(fmaxf(top, x[j]), x[j + 1]);
            const float next = fmaxf(ref, top), base = next == -INFINITY ? 0.f : next;
            const float off = -base * a.down;
            const uint64_t cc = f2_pack(a.c, a.c), down = f2_pack(a.down, a.down), minus = f2_pack(off, off);
            uint64_t part[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
            for (int j = 0; j < CE_PART; j += 2) {
                const uint64_t pair = f2_pack(x[j], x[j + 1]);
                float e0, e1;
                f2_unpack(BIAS ? f2_add(pair, minus) : f2_mul(f2_fma(pair, down, minus), cc), e0, e1);
                part[j / 2 & 3] = f2_add(part[j / 2 & 3], f2_pack(ce_exp2(e0), ce_exp2(e1)));
            }
            float lo, hi;
            f2_unpack(f2_add(f2_add(part[0], part[1]), f2_add(part[2], part[3])), lo, hi);
            sum = fmaf(sum, ce_exp2(BIAS ? ref - base : fmaf(ref, a.down, off) * a.c), lo + hi);
            ref = next;
        }
        __device__ __forceinline__ void segment(const CeScoreArgs& a, bool first, uint32_t taddr, bool live) {
            if (!idle) CeSums<SEGMENTS, TILE == CE_SMALL>::segment(a, first, taddr, live);
        }
        template <typename D>
        __device__ __forceinline__ void tile(const CeScoreArgs& a, const CeUnit& u, int t, uint32_t taddr, bool live, bool more, D&& done) {
            if (idle) {  // no query is behind the warp's lanes
                done();
                return;
            }
            const int n0 = a.n0 + (u.tile0 + t) * BN + group * CE_PART, left = a.n1 - n0, at = target - n0;
            if (BIAS) ce_bias_tile(a.bias, n0, a.n1, s_bias, lane);
            this->read(a, taddr, live, more, [&](float (&x)[CE_PART]) {
            done();
            if (left < CE_PART || __any_sync(0xFFFFFFFFu, (unsigned)at < (unsigned)CE_PART)) {  // seldom
                float v = 0.f;
#pragma unroll
                for (int j = 0; j < CE_PART; ++j) {
                    if (j == at) v = x[j];
                    if (!BIAS && j >= left) x[j] = -INFINITY;
                }
                if ((unsigned)at < (unsigned)CE_PART) a.target_scores[q] = v;
            }
            if (BIAS) {
#pragma unroll
                for (int j = 0; j < CE_PART; ++j) {  // a row that is masked may hold anything
                    const float b = s_bias[j];
                    x[j] = b == -INFINITY ? b : fmaf(x[j], a.c, b);
                }
            }
            add(a, x);
            if (!live) sum = __int_as_float(0x7FFFFFFF);
            });
        }
        __device__ __forceinline__ void unit_end(const CeScoreArgs& a, const CeUnit& u) {
            if (q < a.m) a.partial[(int64_t)q * a.slots + u.block * (BN / CE_PART) + group] = make_float2(ref, sum);
        }
    };
};

// G of a piece, 128 neighbouring bytes of a query to a thread.  4,099 x 6,656 x 2,048 float16 102 us, 1,095 TFLOP/s (in one sum over K 82; see CE_SEGMENT).
template <int PLANES, bool BIAS, bool HALF, bool SEGMENTS, int TILE>
struct CeGradPolicy : CeScoreBase<PLANES, SEGMENTS, TILE> {
    static constexpr int BN = CeScoreBase<PLANES, SEGMENTS, TILE>::BN;
    struct Epilogue : CeSums<SEGMENTS, TILE == CE_SMALL> {
        int q, quarter, group, lane, rank, target;
        bool idle;
        float term, factor;
        float* s_bias;
        __device__ __forceinline__ Epilogue(const CeScoreArgs&, unsigned char* smem, int warp, int quarter_, int group_, int lane_, int rank_)
            : quarter(quarter_), group(group_), lane(lane_), rank(rank_), s_bias(reinterpret_cast<float*>(smem) + warp * CE_PART) {}
        __device__ __forceinline__ void unit_begin(const CeScoreArgs& a, const CeUnit& u) {
            q = u.m0 + rank * TG_M + quarter * 32 + lane;
            idle = q - lane >= a.m;
            const bool in = q < a.m;
            term = in ? __ldcg(a.terms + q) : 0.f;
            factor = in ? __ldcg(a.factors + q) : 0.f;
            target = in ? __ldcg(a.target_cols + q) : -1;
            if (HALF) factor = ldexpf(factor, ce_scale_exponent(a.amax) - a.shift);
        }
        __device__ __forceinline__ void segment(const CeScoreArgs& a, bool first, uint32_t taddr, bool live) {
            if (!idle) CeSums<SEGMENTS, TILE == CE_SMALL>::segment(a, first, taddr, live);
        }
        template <typename D>
        __device__ __forceinline__ void tile(const CeScoreArgs& a, const CeUnit& u, int t, uint32_t taddr, bool live, bool more, D&& done) {
            if (idle) {  // no query is behind the warp's lanes
                done();
                return;
            }
            const int first = (u.tile0 + t) * BN + group * CE_PART, n0 = a.n0 + first, left = a.n1 - n0, at = target - n0;
            if (BIAS) ce_bias_tile(a.bias, n0, a.n1, s_bias, lane);
            this->read(a, taddr, live, more, [&](float (&x)[CE_PART]) {
            done();
            if (!live) factor = __int_as_float(0x7FFFFFFF);
#pragma unroll
            for (int j = 0; j < CE_PART; ++j) x[j] = ce_exp2(BIAS ? fmaf(x[j], a.c, s_bias[j]) + term : fmaf(x[j], a.c, term)) * factor;  // as in the losses' pass: the bias first
            if (left < CE_PART || __any_sync(0xFFFFFFFFu, (unsigned)at < (unsigned)CE_PART)) {  // seldom; behind the last row G has zeros
#pragma unroll
                for (int j = 0; j < CE_PART; ++j)
                    if (j == at || j >= left) x[j] = 0.f;
            }
            if (q >= a.m) return;
            uint16_t* const out = reinterpret_cast<uint16_t*>(a.G) + (int64_t)q * a.pitch + first;
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
                uint4* const o = reinterpret_cast<uint4*>(out + p * a.plane);
#pragma unroll
                for (int i = 0; i < CE_PART / 8; ++i) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float &lo = x[8 * i + 2 * k], &hi = x[8 * i + 2 * k + 1];
                        if (HALF) {
                            w[k] = pack_scores(static_cast<const __half*>(nullptr), lo, hi);
                        } else {
                            w[k] = pack_scores(static_cast<const __nv_bfloat16*>(nullptr), lo, hi);
                            if (p + 1 < PLANES) lo -= __uint_as_float(w[k] << 16), hi -= __uint_as_float(w[k] & 0xFFFF0000u);
                        }
                    }
                    o[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            });
        }
        __device__ __forceinline__ void unit_end(const CeScoreArgs&, const CeUnit&) {}
    };
};

// Bound by the tensor pipe and by the ends of the few waves: 6,656 x 2,048 by 4,099 88 us, 4,099 x 2,048 by 6,656 97.
// Products with G: out[split][row][col] (+)= sum over a split of K of A's row by B's column.
struct CeProductArgs {
    int* d_error;
    unsigned units;
    uint32_t idesc;
    int rows, cols;
    int b0;                   // entry of K that B begins with
    int kb, kper;             // steps of K, and as many in a split
    int tiles_m, tiles_n, m_tile;
    bool accumulate;
    float* out;
    // dX from sums that are complete: 16-bit values with the targets' part, over the temperature
    void* typed;
    int64_t ld;
    const uint32_t* amax;
    const int* where;
    int own_splits;
    int64_t where_stride;
    const float* sums;
    float inv_t;
};
struct CeProductUnit {
    static constexpr int tiles = 1;
    int m0, nt, k0, k1, split;
    __device__ __forceinline__ CeProductUnit(const CeProductArgs& a, unsigned u) {
        const int mt = (int)(u % (unsigned)a.tiles_m);
        u /= (unsigned)a.tiles_m;
        nt = (int)(u % (unsigned)a.tiles_n);
        split = (int)(u / (unsigned)a.tiles_n);
        m0 = mt * a.m_tile;
        k0 = split * a.kper, k1 = min(a.kb, k0 + a.kper);
    }
};
// 32 columns of a row of dX from `col` on, times `scale`, with the targets' part.
__device__ __forceinline__ void ce_with_own(const CeProductArgs& a, int row, int col, float scale, uint32_t taddr, bool live, float (&v)[32]) {
    uint32_t r[32];
    tg_read(taddr, live, r);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) * scale;
    ce_add_own(v, a.where + row, a.where_stride, row < a.rows ? a.own_splits : 0, a.sums, a.cols, col, a.inv_t);
}
template <typename T>
__device__ __noinline__ void ce_store_turned(const CeProductArgs& a, int row, int lane, int col, float scale, uint32_t taddr, bool live) {
    float v[32];
    ce_with_own(a, row, col, scale, taddr, live, v);
    ce_turn(v, lane);
    T* const to = reinterpret_cast<T*>(a.typed) + (int64_t)(row - lane) * a.ld + col + lane;
    if (col + lane < a.cols) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (row - lane + j < a.rows) store_score(to + j * a.ld, v[j]);
    }
}
// N columns of a row of dX from column col0 on.
template <typename T, int N>
__device__ __forceinline__ void ce_store_typed(const CeProductArgs& a, int row, int lane, int col0, uint32_t taddr, bool live) {
    constexpr int V = 16 / sizeof(T);
    const float scale = std::is_same<T, __half>::value ? ce_scale_back(a.inv_t, ce_scale_exponent(a.amax)) : a.inv_t;
    if (a.cols % V != 0 || a.ld % V != 0 || ((uintptr_t)a.typed & 15) != 0) {  // no 16 bytes of a row lie together: rows turned, so that neighbouring lanes have neighbouring columns
        for (int c0 = 0; c0 < N && col0 + c0 < a.cols; c0 += 32) ce_store_turned<T>(a, row, lane, col0 + c0, scale, taddr + c0, live);
        return;
    }
    T* const o = reinterpret_cast<T*>(a.typed) + (int64_t)row * a.ld + col0;
#pragma unroll 1
    for (int c0 = 0; c0 < N && col0 + c0 < a.cols; c0 += 32) {
        float v[32];
        ce_with_own(a, row, col0 + c0, scale, taddr + c0, live, v);
#pragma unroll
        for (int j = 0; j < 32; j += V) {
            if (row >= a.rows || col0 + c0 + j >= a.cols) break;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4*>(o + c0 + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            } else {
                const T* const t = nullptr;
                *reinterpret_cast<uint4*>(o + c0 + j) =
                    make_uint4(pack_scores(t, v[j], v[j + 1]), pack_scores(t, v[j + 2], v[j + 3]), pack_scores(t, v[j + 4], v[j + 5]), pack_scores(t, v[j + 6], v[j + 7]));
            }
        }
    }
}
// TYPED: 0: sums in 32 bits; 1, 2, 3: results in bfloat16, float16, float32.
template <int PLANES, bool AMN, int N, bool PAIRS, int TYPED>
struct CeProductPolicy {
    static constexpr bool A_MN = AMN, B_MN = true, I8 = false, PARTS = true, PAIR = PAIRS;
    static constexpr int BN = N, SEGMENTS = 0, EPI_BYTES = 0, EPI_WARPS = 8;
    using Pairs = PlanePairs<PLANES>;
    using Args = CeProductArgs;
    using Unit = CeProductUnit;
    static __device__ __forceinline__ void load(const Args& a, const Unit& u, int, int pa, int pb, int k, const CUtensorMap* ta, const CUtensorMap* tb, unsigned char* sa,
                                                unsigned char* sb, uint32_t bar, int rank) {
        const int m0 = u.m0 + rank * TG_M;
        if (AMN) {
            tma_load_3d<PAIR>(sa, ta, bar, m0, k * 64, pa);
            tma_load_3d<PAIR>(sa + TG_BOX_BYTES, ta, bar, m0 + 64, k * 64, pa);
        } else {
            tma_load_3d<PAIR>(sa, ta, bar, k * 64, m0, pa);
        }
        constexpr int HERE = BN / (PAIR ? 2 : 1);
#pragma unroll
        for (int i = 0; i < HERE / 64; ++i) tma_load_3d<PAIR>(sb + i * TG_BOX_BYTES, tb, bar, u.nt * BN + rank * HERE + i * 64, a.b0 + k * 64, pb);
    }
    static __device__ __forceinline__ int n_mma(const Args& a, const Unit& u, int) { return min(BN, (a.cols - u.nt * BN + 15) & ~15); }

    struct Epilogue {
        int quarter, group, lane, rank;
        __device__ __forceinline__ Epilogue(const Args&, unsigned char*, int, int quarter_, int group_, int lane_, int rank_)
            : quarter(quarter_), group(group_), lane(lane_), rank(rank_) {}
        __device__ __forceinline__ void unit_begin(const Args&, const Unit&) {}
        __device__ __forceinline__ void unit_end(const Args&, const Unit&) {}
        template <typename D>
        __device__ __forceinline__ void tile(const Args& a, const Unit& u, int, uint32_t taddr, bool live, bool, D&& done) {
            const int row = u.m0 + rank * TG_M + quarter * 32 + lane;
            if (row - lane >= a.rows) {
                done();
                return;
            }
            if constexpr (TYPED != 0) {
                ce_store_typed<std::conditional_t<TYPED == 3, float, std::conditional_t<TYPED == 2, __half, __nv_bfloat16>>, BN / 2>(a, row, lane, u.nt * BN + group * (BN / 2), taddr, live);
                done();
                return;
            }
            float* const out = a.out + ((int64_t)u.split * a.rows + row) * a.cols + u.nt * BN + group * (BN / 2);
            const int width = min(BN / 2, a.cols - u.nt * BN - group * (BN / 2));
            const bool wide = (a.cols & 3) == 0;
#pragma unroll 1
            for (int c0 = 0; c0 < width; c0 += 32) {
                uint32_t r[32];
                tg_read(taddr + c0, live, r);
                if (wide) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (row >= a.rows || c0 + j >= width) break;
                        float4 v = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
                        float4* const o = reinterpret_cast<float4*>(out + c0 + j);
                        if (a.accumulate) {
                            const float4 w = __ldcg(o);
                            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                        }
                        *o = v;
                    }
                } else {
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
                    ce_turn(v, lane);
                    float* const column = out - (int64_t)lane * a.cols + c0 + lane;
                    if (c0 + lane < width) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (row - lane + j < a.rows) column[(int64_t)j * a.cols] = v[j] + (a.accumulate ? __ldcg(column + (int64_t)j * a.cols) : 0.f);
                    }
                }
            }
            done();
        }
    };
};

// Losses of up to 16 queries in 32 bits, which would leave the tensor cores' lanes empty and cost the planes' reads and writes: bound by reading the rows once.  A thread has a row, 32 columns of
// 256 rows at a time come through shared memory; the queries' values are read from there by all lanes at once.  Maxima and sums are a thread's until the end.
// Where it is taken, on the tensor cores | here (us): losses of 500,000 x 16, 1 query 126 | 24, 16 of them 129 | 82; 128,000 x 500, 1 query 297 | 83, but 16 of 2,000 x 500 29 | 85.  Gradients of
// 500,000 x 128, 1 query 660 | 279, 16 of them 621 | 461, of 2,000 x 128 44 | 50, but of 8,000 x 500 81 | 159.  16 bits are none the better for it (500,000 x 128, 4 queries 229 | 439).
constexpr int CE_FEW_LOSS = 1024, CE_FEW_GRAD = 192;  // queries by columns; columns
constexpr int CE_FEW = 16, CE_FEW_COLS = 32, CE_FEW_THREADS = 256;
template <int M, bool BIAS>
__global__ void __launch_bounds__(CE_FEW_THREADS, 2) ce_few_kernel(const float* __restrict__ Q, int64_t ldq, const float* __restrict__ X, int64_t ldx, int m, int n, int d,
                                                                const float* __restrict__ bias, float c, float down, const int64_t* __restrict__ targets, float2* __restrict__ partial,
                                                                float* __restrict__ target_scores, KernelBefore before) {
    behind_kernel_before(Q, X, bias, targets, partial, target_scores, before);
    __shared__ float s_x[CE_FEW_COLS][CE_FEW_THREADS + 1];
    __shared__ alignas(16) float s_q[CE_FEW_COLS][M < 4 ? 4 : M];
    __shared__ float2 s_part[CE_FEW_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float by = BIAS ? 1.f : c;
    float ref[M], sum[M];
    int target[M];
#pragma unroll
    for (int q = 0; q < M; ++q) {
        const int64_t t = q < m && targets ? __ldcg(targets + q) : -1;
        target[q] = t < 0 || t >= n ? -1 : (int)t;
        ref[q] = -INFINITY, sum[q] = 0.f;
    }
    for (int64_t row0 = (int64_t)blockIdx.x * CE_FEW_THREADS; row0 < n; row0 += (int64_t)gridDim.x * CE_FEW_THREADS) {
        float acc[M] = {};
        for (int c0 = 0; c0 < d; c0 += CE_FEW_COLS) {
            float v[CE_FEW_COLS];  // a warp's 32 rows, a column to a lane
#pragma unroll
            for (int j = 0; j < CE_FEW_COLS; ++j) {
                const int64_t row = row0 + warp * 32 + j;
                v[j] = row < n && c0 + lane < d ? __ldcg(X + row * ldx + c0 + lane) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CE_FEW_COLS; ++j) s_x[lane][warp * 32 + j] = v[j];
            for (int i = threadIdx.x; i < CE_FEW_COLS * M; i += CE_FEW_THREADS) {
                const int q = i / CE_FEW_COLS, k = i % CE_FEW_COLS;
                s_q[k][q] = q < m && c0 + k < d ? __ldcg(Q + q * ldq + c0 + k) : 0.f;
            }
            __syncthreads();
            float part[M] = {};  // sums of sums: single ones leave losses of one query by 8,962 x 412 an error of 1.1e-6, these 2.0e-7
#pragma unroll 8
            for (int k = 0; k < min(CE_FEW_COLS, d - c0); ++k) {
                const float x = s_x[k][threadIdx.x];
#pragma unroll
                for (int q = 0; q < M; ++q) part[q] = fmaf(s_q[k][q], x, part[q]);
            }
#pragma unroll
            for (int q = 0; q < M; ++q) acc[q] += part[q];
        }
        const int64_t row = row0 + threadIdx.x;
        if (row < n) {
            const float b = BIAS ? __ldcg(bias + row) * CE_LOG2E : 0.f;
#pragma unroll
            for (int q = 0; q < M; ++q) {
                if (target[q] == row) target_scores[q] = acc[q];
                const float z = !BIAS ? acc[q] : b == -INFINITY ? b : fmaf(acc[q], c, b), next = fmaxf(ref[q], z), off = next == -INFINITY ? 0.f : -next * down;
                sum[q] = fmaf(sum[q], ce_exp2(fmaf(ref[q], down, off) * by), ce_exp2(fmaf(z, down, off) * by));
                ref[q] = next;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < M; ++q) {
        if (q >= m) break;
        float top = ref[q];
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float all = sum[q] * ce_exp2(fmaf(ref[q], down, top == -INFINITY ? 0.f : -top * down) * by);
        for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
        __syncthreads();
        if (lane == 0) s_part[warp] = make_float2(top, all);
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < CE_FEW_THREADS / 32; ++w) top = fmaxf(top, s_part[w].x);
            const float off = top == -INFINITY ? 0.f : -top * down;
            all = 0.f;
            for (int w = 0; w < CE_FEW_THREADS / 32; ++w) all = fmaf(s_part[w].y, ce_exp2(fmaf(s_part[w].x, down, off) * by), all);
            partial[(int64_t)q * gridDim.x + blockIdx.x] = make_float2(top, all);
        }
    }
}

// Gradients of up to 16 queries, likewise.  First the scores of 256 rows, a row to a thread, and G, to which the target's own coefficient belongs here (nothing is rounded to 16 bits); then, a
// column to a lane, what the rows put into dQ, and dX.  dQ's sums are a CTA's, in shared memory; ce_finish_kernel adds them up.
template <typename T, int M, bool BIAS>
__global__ void __launch_bounds__(CE_FEW_THREADS, 2) ce_few_grad_kernel(const T* __restrict__ Q, int64_t ldq, const T* __restrict__ X, int64_t ldx, int m, int n, int d,
                                                                        const float* __restrict__ bias, float c, float inv_t, const float* __restrict__ terms,
                                                                        const float* __restrict__ factors, const float* __restrict__ own, const int* __restrict__ cols,
                                                                        float* __restrict__ parts, T* __restrict__ dX, int64_t ldo, KernelBefore before) {
    behind_kernel_before(Q, X, bias, terms, factors, own, cols, parts, dX, before);
    constexpr int MQ = M < 4 ? 4 : M;
    __shared__ alignas(16) float s_x[CE_FEW_COLS][CE_FEW_THREADS + 1];
    __shared__ alignas(16) float s_q[CE_FEW_COLS][MQ];
    extern __shared__ float s_sums[];  // [m][d]
    float* const s_add = &s_x[0][0];   // [warp][query][column of 32], where the rows' values are no longer needed
    float(*const s_g)[MQ] = reinterpret_cast<float(*)[MQ]>(s_add + CE_FEW_THREADS * M);
    static_assert(CE_FEW_THREADS * (M + MQ) <= CE_FEW_COLS * (CE_FEW_THREADS + 1), "");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; parts && i < m * d; i += CE_FEW_THREADS) s_sums[i] = 0.f;
    for (int64_t row0 = (int64_t)blockIdx.x * CE_FEW_THREADS; row0 < n; row0 += (int64_t)gridDim.x * CE_FEW_THREADS) {
        float acc[M] = {};
        for (int c0 = 0; c0 < d; c0 += CE_FEW_COLS) {
            float v[CE_FEW_COLS];  // a warp's 32 rows, a column to a lane
#pragma unroll
            for (int j = 0; j < CE_FEW_COLS; ++j) {
                const int64_t row = row0 + warp * 32 + j;
                v[j] = row < n && c0 + lane < d ? ce_float(__ldcg(X + row * ldx + c0 + lane)) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CE_FEW_COLS; ++j) s_x[lane][warp * 32 + j] = v[j];
            for (int i = threadIdx.x; i < CE_FEW_COLS * M; i += CE_FEW_THREADS) {
                const int q = i / CE_FEW_COLS, k = i % CE_FEW_COLS;
                s_q[k][q] = q < m && c0 + k < d ? ce_float(__ldcg(Q + q * ldq + c0 + k)) : 0.f;
            }
            __syncthreads();
            float part[M] = {};  // sums of sums: single ones leave losses of one query by 8,962 x 412 an error of 1.1e-6, these 2.0e-7
#pragma unroll 8
            for (int k = 0; k < min(CE_FEW_COLS, d - c0); ++k) {
                const float x = s_x[k][threadIdx.x];
#pragma unroll
                for (int q = 0; q < M; ++q) part[q] = fmaf(s_q[k][q], x, part[q]);
            }
#pragma unroll
            for (int q = 0; q < M; ++q) acc[q] += part[q];
        }
        __syncthreads();
        const int64_t row = row0 + threadIdx.x;
        const float b = BIAS && row < n ? __ldcg(bias + row) * CE_LOG2E : 0.f;
        const bool masked = row >= n || (BIAS && b == -INFINITY);
#pragma unroll
        for (int q = 0; q < M; ++q) {
            float g = 0.f;
            if (q < m && !masked) {
                const float term = __ldcg(terms + q);
                g = __ldcg(cols + q) == row ? __ldcg(own + q) : ce_exp2(BIAS ? fmaf(acc[q], c, b) + term : fmaf(acc[q], c, term)) * __ldcg(factors + q);
            }
            s_g[threadIdx.x][q] = g;
        }
        const unsigned live = __ballot_sync(0xFFFFFFFFu, !masked);  // a row that is masked may hold anything
        for (int c0 = 0; c0 < d; c0 += CE_FEW_COLS) {
            const int col = c0 + lane;
            float q_of[M], sum[M] = {};
#pragma unroll
            for (int q = 0; q < M; ++q) q_of[q] = dX && q < m && col < d ? ce_float(__ldcg(Q + q * ldq + col)) : 0.f;
            __syncwarp();
#pragma unroll 4
            for (int j = 0; j < 32; ++j) {
                const int64_t at = row0 + warp * 32 + j;
                const float x = parts && live >> j & 1u && col < d ? ce_float(__ldcg(X + at * ldx + col)) : 0.f;
                float out = 0.f;
#pragma unroll
                for (int q = 0; q < M; ++q) {
                    const float g = s_g[warp * 32 + j][q];
                    sum[q] = fmaf(g, x, sum[q]);
                    out = fmaf(g, q_of[q], out);
                }
                if (dX && at < n && col < d) dX[at * ldo + col] = (T)(out * inv_t);
            }
            if (parts) {
                __syncthreads();
#pragma unroll
                for (int q = 0; q < M; ++q) s_add[(warp * M + q) * 32 + lane] = sum[q];
                __syncthreads();
                for (int i = threadIdx.x; i < 32 * M; i += CE_FEW_THREADS) {
                    const int q = i / 32, k = i % 32;
                    float all = 0.f;
                    for (int w = 0; w < CE_FEW_THREADS / 32; ++w) all += s_add[(w * M + q) * 32 + k];
                    if (q < m && c0 + k < d) s_sums[q * d + c0 + k] += all;
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; parts && i < m * d; i += CE_FEW_THREADS) parts[(int64_t)blockIdx.x * m * d + i] = s_sums[i];
}

// ---- what the products need beforehand: one launch, whose CTAs have a share of one of five jobs each --------------------------------------------------------------------
struct CePlanes {  // of a matrix
    const void* from;
    int64_t ld, rows;
    const float* bias;
    uint16_t* to;
    bool wide;  // rows begin at multiples of 16 bytes
};
struct CePrepare {
    unsigned ends[5];         // CTAs up to the end of each job: planes of Q, of X, the bias, the queries' terms, the targets' sums
    int m, n, d, pitch, own_rows, own_tiles, own_shares, own_cols, own_queries;
    CePlanes planes[2];
    const float* bias;
    float* bias2;
    const float *losses, *lse, *lse_low, *grad_losses, *grad_lse;
    const int64_t* targets;
    float *terms, *factors, *own, *sums;
    int *cols, *where;
    int shift, t_shift;
    bool lines;               // terms, factors and cols in lines of 128
    uint32_t* amax;
    const void* Q;
    int64_t ldq;
};
// A matrix as planes of 16 bits with rows of `pitch` entries, zeros behind a row's end: three bfloat16 that sum up to each float, or the values as they are.  Rows that the bias masks become
// zeros: G has zeros for them, and what they hold may not be finite.
template <typename T, int PLANES>
__device__ __forceinline__ void ce_planes_part(const CePrepare& a, const CePlanes& p, unsigned block) {
    const int each = a.pitch / 8;  // eight columns to a thread
    const int64_t i = (int64_t)block * 256 + threadIdx.x, total = p.rows * each;
    if (i >= total) return;
    const int64_t row = total >> 32 ? i / each : (int64_t)((uint32_t)i / (uint32_t)each);
    const int col = (int)(i - row * each) * 8;
    const T* const x = static_cast<const T*>(p.from) + row * p.ld + col;
    const bool some = !(p.bias && p.bias[row] == -INFINITY);
    alignas(16) T v[8];
    if (some && p.wide && col + 8 <= a.d) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(v)[k] = reinterpret_cast<const uint4*>(x)[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = some && col + k < a.d ? x[k] : (T)0.f;
    }
    uint4* const o = reinterpret_cast<uint4*>(p.to) + i;
    if constexpr (PLANES == 1) {
        *o = *reinterpret_cast<const uint4*>(v);
    } else {
#pragma unroll
        for (int k = 0; k < PLANES; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = pack_scores(static_cast<const __nv_bfloat16*>(nullptr), v[2 * j], v[2 * j + 1]);
                v[2 * j] -= __uint_as_float(w[j] << 16);
                v[2 * j + 1] -= __uint_as_float(w[j] & 0xFFFF0000u);
            }
            o[k * total] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
__device__ __forceinline__ void ce_bias_part(const CePrepare& a, unsigned block) {
    const int i = block * 256 + threadIdx.x;
    if (i < a.n) a.bias2[i] = a.bias[i] * CE_LOG2E;
    else if (i < ((a.n + 127) & ~127)) a.bias2[i] = 0.f;
}

// WARPS warps join a query's blocks.
template <int WARPS>
__global__ void __launch_bounds__(256) ce_join_kernel(const float2* __restrict__ partial, int slots, int m, int n, const int64_t* __restrict__ targets,
                                                      const float* __restrict__ target_scores, const float* __restrict__ bias2, float c, float down, float* __restrict__ losses,
                                                      float* __restrict__ lse, float* __restrict__ lse_low, KernelBefore before) {
    behind_kernel_before(partial, targets, target_scores, bias2, losses, lse, lse_low, before);
    __shared__ float s_top[8];
    __shared__ double s_sum[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = blockIdx.x * (8 / WARPS) + warp / WARPS, first = (warp % WARPS) * 32 + lane;
    const float2* const p = partial + (int64_t)min(q, m - 1) * slots;
    float top = -INFINITY;
#pragma unroll 8
    for (int i = first; i < slots; i += 32 * WARPS) top = fmaxf(top, __ldcg(p + i).x);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (WARPS > 1) {
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_top[warp / WARPS * WARPS + w]);
    }
    const float base = top == -INFINITY ? 0.f : top * down, by = bias2 ? 1.f : c;  // scores, or exponents
    double sum = 0.;
#pragma unroll 8
    for (int i = first; i < slots; i += 32 * WARPS) {
        const float2 v = __ldcg(p + i);
        sum += (double)v.y * (double)exp2f(fmaf(v.x, down, -base) * by);
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (WARPS > 1) {
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        sum = 0.;
        for (int w = 0; w < WARPS; ++w) sum += s_sum[warp / WARPS * WARPS + w];
    }
    if (first || q >= m) return;
    const double ln2 = 0.69314718055994530942, two = (double)base * (double)by + log2(sum), whole = two * ln2;
    const float high = (float)whole;
    lse[q] = high;
    lse_low[q] = isfinite(high) ? (float)(whole - (double)high) : 0.f;
    float loss = 0.f;
    const int64_t t = targets ? __ldcg(targets + q) : -1;
    if (t >= 0 && t < n) {
        const float b = bias2 ? __ldcg(bias2 + t) : 0.f, s = __ldcg(target_scores + q);
        const double z = b == -INFINITY ? (double)b : bias2 ? (double)fmaf(s, c, b) : (double)(s * down) * (double)c;  // as in the sums
        loss = z == -INFINITY && two == two ? INFINITY : (float)((two - z) * ln2);
        if (loss < 0.f) loss = 0.f;
    }
    losses[q] = loss;
}

// The target of a query that has a loss to go by, or -1; and what its own entry puts into the gradients.
__device__ __forceinline__ int ce_target(const CePrepare& a, int q) {
    const int64_t t = a.targets ? a.targets[q] : -1;
    return t >= 0 && t < a.n && a.losses[q] < INFINITY ? (int)t : -1;
}
__device__ __forceinline__ float ce_own(const CePrepare& a, int q) {
    const float loss = a.losses[q], g = a.grad_losses ? a.grad_losses[q] : 0.f, e = a.grad_lse ? a.grad_lse[q] : 0.f;
    return ldexpf(g * expm1f(-loss) + e * expf(-loss), -a.t_shift);
}
__device__ __forceinline__ void ce_terms_part(const CePrepare& a, unsigned block) {
    const int q = block * 256 + threadIdx.x;
    if (q >= a.m) {
        if (a.lines && q < ((a.m + 127) & ~127)) a.terms[q] = -INFINITY, a.factors[q] = 0.f, a.cols[q] = -1;
        return;
    }
    const double two = ((double)a.lse[q] + (double)a.lse_low[q]) * 1.4426950408889634074 - (double)a.shift;
    const float high = (float)two;
    const bool none = high == -INFINITY;
    const int t = ce_target(a, q);
    const float g = t >= 0 && a.grad_losses ? a.grad_losses[q] : 0.f, e = a.grad_lse ? a.grad_lse[q] : 0.f;
    a.terms[q] = none ? -INFINITY : -high;
    const float f = ldexpf((g + e) * (isfinite(high) ? (float)exp2(-(two - (double)high)) : 1.f), -a.t_shift);
    a.factors[q] = f;
    a.cols[q] = t;
    a.own[q] = t >= 0 ? ce_own(a, q) : 0.f;
    if (a.amax && isfinite(f)) atomicMax(a.amax, __float_as_uint(fabsf(f)));
}

// Sums over the queries whose target is a row, own[i] q_i: sums[first query of the row][d], and which one that is for each row (-1: none); of few rows for each of own_queries queries.  A CTA takes own_rows rows, or own_cols columns of
// them, and looks through all targets; they come in ascending order.
constexpr int CE_OWN_ROWS = 1024, CE_OWN_LIST = 2560, CE_OWN_COLS = 8, CE_OWN_AHEAD = 5;  // rows at most; entries; columns of a lane at a time; targets of a thread
template <typename T>
__device__ __forceinline__ void ce_own_part(const CePrepare& a, unsigned block) {
    __shared__ int s_first[CE_OWN_ROWS];
    __shared__ int s_query[CE_OWN_LIST];
    __shared__ float s_own[CE_OWN_LIST];
    __shared__ uint16_t s_row[CE_OWN_LIST];
    __shared__ unsigned s_hits[CE_OWN_AHEAD * 8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned share = block % (unsigned)a.own_shares, tile = block / (unsigned)a.own_shares % (unsigned)a.own_tiles, split = block / (unsigned)a.own_shares / (unsigned)a.own_tiles;
    const int64_t row0 = (int64_t)tile * a.own_rows, q0 = (int64_t)split * a.own_queries, q1 = min((int64_t)a.m, q0 + a.own_queries);
    const int first_col = (int)share * a.own_cols, last_col = min(a.d, first_col + a.own_cols);
    const T* const Q = static_cast<const T*>(a.Q);
    for (int r = threadIdx.x; r < a.own_rows; r += 256) s_first[r] = -1;
    int held = 0;  // the same for all threads
    constexpr int STEP = CE_OWN_AHEAD * 256;
    for (int64_t i0 = q0; i0 < q1; i0 += STEP) {
        int64_t of[CE_OWN_AHEAD];
        bool any = false;
#pragma unroll
        for (int k = 0; k < CE_OWN_AHEAD; ++k) {
            const int64_t i = i0 + k * 256 + threadIdx.x, r = (a.targets && i < q1 ? a.targets[i] : -1) - row0;
            of[k] = r >= 0 && r < a.own_rows && r + row0 < a.n && a.losses[i] < INFINITY ? r : -1;
            const unsigned hits = __ballot_sync(0xFFFFFFFFu, of[k] >= 0);
            if (lane == 0) s_hits[k * 8 + warp] = hits;
            any = any || of[k] >= 0;
        }
        if (__syncthreads_or(any)) {
#pragma unroll
            for (int k = 0; k < CE_OWN_AHEAD; ++k)
                for (int w = 0; w < 8; ++w) {
                    const unsigned hits = s_hits[k * 8 + w];
                    if (w == warp && of[k] >= 0) {
                        const int at = held + __popc(hits & ((1u << lane) - 1u));
                        s_query[at] = (int)i0 + k * 256 + threadIdx.x;
                        s_row[at] = (uint16_t)of[k];
                    }
                    held += __popc(hits);
                }
            __syncthreads();
        }
        if (held && (held + STEP > CE_OWN_LIST || i0 + STEP >= q1)) {
            for (int e = threadIdx.x; e < held; e += 256) s_own[e] = ce_own(a, s_query[e]);
            __syncthreads();
            for (int e = warp; e < held; e += 8) {  // a warp takes an entry, if it is the first of its row, with those that follow
                const int rr = s_row[e];
                bool first = true;
                for (int e0 = 0; e0 < e && first; e0 += 32) first = !__any_sync(0xFFFFFFFFu, e0 + lane < e && s_row[e0 + lane] == rr);
                if (!first) continue;
                const bool fresh = s_first[rr] < 0;
                const int slot = fresh ? s_query[e] : s_first[rr];
                auto columns = [&](auto of_lane) {
                    constexpr int COLS = decltype(of_lane)::value, BATCH = 32 / COLS;  // 32 loads in flight
                    for (int c0 = first_col; c0 < last_col; c0 += 32 * COLS) {
                        float acc[COLS] = {};
                        int e0 = e & ~31;
                        unsigned b = __ballot_sync(0xFFFFFFFFu, e0 + lane < held && s_row[e0 + lane] == rr);
                        while (e0 < held) {
                            float f[BATCH], v[BATCH][COLS];
                            unsigned real = 0;
#pragma unroll
                            for (int h = 0; h < BATCH; ++h) {  // the next entries of the row
                                while (!b && e0 < held) {
                                    e0 += 32;
                                    b = __ballot_sync(0xFFFFFFFFu, e0 + lane < held && s_row[e0 + lane] == rr);
                                }
                                const int at = b ? e0 + __ffs(b) - 1 : 0;
                                real |= (b != 0u) << h;
                                const T* const from = Q + (int64_t)s_query[at] * a.ldq + c0 + lane;
                                f[h] = s_own[at];
#pragma unroll
                                for (int k = 0; k < COLS; ++k) v[h][k] = b && c0 + k * 32 + lane < a.d ? ce_float(from[k * 32]) : 0.f;
                                b &= b - 1u;
                            }
#pragma unroll
                            for (int h = 0; h < BATCH; ++h)
#pragma unroll
                                for (int k = 0; k < COLS; ++k)
                                    if (real >> h & 1u) acc[k] = fmaf(f[h], v[h][k], acc[k]);
                        }
#pragma unroll
                        for (int k = 0; k < COLS; ++k) {
                            const int col = c0 + k * 32 + lane;
                            if (col < a.d) {
                                float* const s = a.sums + (int64_t)slot * a.d + col;
                                *s = fresh ? acc[k] : *s + acc[k];
                            }
                        }
                    }
                };
                if (last_col - first_col > 64) columns(std::integral_constant<int, CE_OWN_COLS>());
                else columns(std::integral_constant<int, 2>());
                __syncwarp();
                if (lane == 0 && fresh) s_first[rr] = slot;
                __syncwarp();
            }
            held = 0;
            __syncthreads();
        }
    }
    __syncthreads();
    if (share == 0)
        for (int r = threadIdx.x; r < a.own_rows && row0 + r < a.n; r += 256) a.where[(int64_t)split * a.n + row0 + r] = s_first[r];
}

template <typename T, int PLANES>
__global__ void __launch_bounds__(256, 4) ce_prepare_kernel(CePrepare a) {
    const unsigned b = blockIdx.x;
    if (b < a.ends[0]) ce_planes_part<T, PLANES>(a, a.planes[0], b);
    else if (b < a.ends[1]) ce_planes_part<T, PLANES>(a, a.planes[1], b - a.ends[0]);
    else if (b < a.ends[2]) ce_bias_part(a, b - a.ends[1]);
    else if (b < a.ends[3]) ce_terms_part(a, b - a.ends[2]);
    else ce_own_part<T>(a, b - a.ends[3]);
}

// Gradients from sums: out[row][col] = (sum over the splits, scaled back, + the target's part) / T.  For queries the target's part is own[row] times the row which[row] of X, for rows
// sums[which[row]].  factors: of the queries, where the sums are of p alone.  One launch for both.
struct CeFinish {
    unsigned blocks;
    const float* parts;
    int splits;
    int64_t split_stride, units;  // units of V columns
    bool wide;                    // V = 4, else 1
    const float* factors;
    const int* which;
    void* out;
    int64_t ldo;
};
struct CeFinishArgs {
    CeFinish rows, queries;
    int d, own_splits;
    int64_t where_stride;
    const uint32_t* amax;
    const float *own, *sums;
    const void* X;
    int64_t ldx;
    float inv_t;
};
template <typename T, bool QUERIES, int V>
__device__ __forceinline__ void ce_finish_part(const CeFinishArgs& a, const CeFinish& f, unsigned block) {
    const int64_t i = (int64_t)block * 256 + threadIdx.x;
    if (i >= f.units) return;
    const unsigned each = (unsigned)a.d / V;
    const int64_t row = f.units >> 32 ? i / each : (int64_t)((uint32_t)i / each);
    const int col = (int)(i - row * each) * V;
    const float* const from = f.parts + row * a.d + col;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
#pragma unroll 4
    for (int s = 0; s < f.splits; ++s) {
        float w[V];
        if (V == 4) *reinterpret_cast<float4*>(w) = __ldcg(reinterpret_cast<const float4*>(from + s * f.split_stride));
        else w[0] = __ldcg(from + s * f.split_stride);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += w[k];
    }
    int w = f.which ? __ldcg(f.which + row) : -1;
    float scale = 1.f;
    if (f.factors) scale = std::is_same<T, __half>::value ? ldexpf(__ldcg(f.factors + row), -CE_HALF_SHIFT) : __ldcg(f.factors + row);
    else if (a.amax) scale = ldexpf(1.f, -ce_scale_exponent(a.amax));
    const float mine = QUERIES && w >= 0 ? __ldcg(a.own + row) : 0.f;
    struct alignas(V * sizeof(T)) Some { T v[V]; };
    Some o;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] *= scale;
    for (int s = 0; s < (QUERIES ? 1 : a.own_splits); ++s) {
        if (s) w = __ldcg(f.which + s * a.where_stride + row);
        if (w < 0) continue;
#pragma unroll
        for (int k = 0; k < V; ++k)
            v[k] += QUERIES ? mine * ce_float(__ldcg(static_cast<const T*>(a.X) + (int64_t)w * a.ldx + col + k)) : __ldcg(a.sums + (int64_t)w * a.d + col + k);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = (T)(v[k] * a.inv_t);
    *reinterpret_cast<Some*>(static_cast<T*>(f.out) + row * f.ldo + col) = o;
}
template <typename T>
__global__ void __launch_bounds__(256) ce_finish_kernel(CeFinishArgs a, KernelBefore before) {
    behind_kernel_before(before);
    const unsigned b = blockIdx.x;
    if (b < a.rows.blocks) {
        if (a.rows.wide) ce_finish_part<T, false, 4>(a, a.rows, b);
        else ce_finish_part<T, false, 1>(a, a.rows, b);
    } else {
        if (a.queries.wide) ce_finish_part<T, true, 4>(a, a.queries, b - a.rows.blocks);
        else ce_finish_part<T, true, 1>(a, a.queries, b - a.rows.blocks);
    }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
struct CeCall {
    CtxPtr c;
    const void *Q, *X;
    int64_t ldq, ldx;
    int type, m, n, d;
    const int64_t* targets;
    const float* bias;
    double temperature;
    int* d_error;
    cudaStream_t stream;
    int planes() const { return type == CULSH_F32 ? 3 : 1; }
    int pitch() const { return (d + 7) & ~7; }
    bool copies(const void* p, int64_t ld) const { return type == CULSH_F32 || !aligned16(p, ld * 2); }
    TgType tg() const { return type == CULSH_F16 ? TG_F16 : TG_BF16; }
    // The losses take differences of scores, without a bias.  They may be beyond float32, and by temperatures beyond 2^100 small again: scores are multiplied by it then, in the same
    // instruction that takes the difference.
    float down() const { return !bias && temperature > 0x1p100 ? 0x1p-64f : 1.f; }
    // Not 0, by which an infinity would be no number: of a temperature beyond 2^149 scores make no difference (at most 2^128 2^-149).
    float c2() const { return std::max((float)(1.4426950408889634 / temperature), 0x1p-149f); }
    // 1 / T as a float of all its bits, times a power of two that the queries' coefficients are less by.
    int t_shift() const { return temperature > 0x1p126 ? std::ilogb(temperature) - 125 : 0; }
    float inv_t() const { return (float)std::ldexp(1 / temperature, t_shift()); }
};

// Pieces of the workspace, each at a multiple of 256 bytes.
struct CeSpace {
    char* base;
    size_t used = 0;
    template <typename T>
    T* take(size_t count) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += (count * sizeof(T) + 255) & ~(size_t)255;
        return p;
    }
};

constexpr size_t CE_G_BYTES = 64u << 20, CE_PARTS_BYTES = 256u << 20;

struct CePlan {
    CeSpace space;
    uint16_t *q_planes = nullptr, *x_planes = nullptr;
    float* bias2 = nullptr;
    // forward
    bool few = false;
    CeTile tile = CE_ONE;
    int block = 0, slots = 0;
    float2* partial = nullptr;
    float* target_scores = nullptr;
    // backward
    float *terms = nullptr, *factors = nullptr, *own = nullptr, *sums = nullptr;
    int *cols = nullptr, *where = nullptr;
    int shift = 0;
    int own_splits = 1;
    uint32_t* amax = nullptr;
    int piece = 0;  // rows
    uint16_t* G = nullptr;
    int splits_q = 0, per_q = 0, splits_x = 0, per_x = 0;
    float *acc_q = nullptr, *parts_x = nullptr;
    bool fused_q = false, fused_x = false;
    int fused_block = 0, fused_block_x = 0;  // tiles of the other side in a unit of dQ, of dX
    int some_q = 0, some_x = 0;              // queries, rows whose sums lie in the workspace at a time

    CePlan(const CeCall& k, bool backward, bool need_q, bool need_x, void* base) : space{static_cast<char*>(base)} {
        const int sms = k.c->sm_count;
        few = !backward && k.type == CULSH_F32 && k.m <= CE_FEW && (int64_t)k.m * k.d <= CE_FEW_LOSS;
        if (few) {
            slots = (int)std::min<size_t>(ceil_div(k.n, CE_FEW_THREADS), (size_t)sms * 3);
            partial = space.take<float2>((size_t)k.m * slots);
            target_scores = space.take<float>(k.m);
            if (k.bias) bias2 = space.take<float>(ceil_div(k.n, 128) * 128);
            return;
        }
        if (backward && k.type == CULSH_F32 && k.m <= CE_FEW && k.d <= CE_FEW_GRAD) {
            few = true;
            terms = space.take<float>(k.m), factors = space.take<float>(k.m), own = space.take<float>(k.m);
            cols = space.take<int>(k.m);
            splits_q = (int)std::min<size_t>(ceil_div(k.n, CE_FEW_THREADS), (size_t)sms * 2);
            if (need_q) acc_q = space.take<float>((size_t)splits_q * k.m * k.d);
            return;
        }
        if (k.copies(k.Q, k.ldq)) q_planes = space.take<uint16_t>((size_t)k.planes() * k.m * k.pitch());
        if (k.copies(k.X, k.ldx) || (backward && k.bias)) x_planes = space.take<uint16_t>((size_t)k.planes() * k.n * k.pitch());
        if (k.bias) bias2 = space.take<float>(ceil_div(k.n, 128) * 128);
        const size_t tiles_q = ceil_div(k.m, TG_M), tiles_n = ceil_div(k.n, CE_BN);
        if (!backward) {
            tile = tile_of(k, k.n);
            const size_t tiles = ceil_div(k.n, tile_rows(tile));
            block = (int)std::max<size_t>(1, std::min<size_t>(16, tiles_q * tiles / ((size_t)sms * 8)));
            auto parts = [&] { return (size_t)(tile_rows(tile) / CE_PART) * ceil_div(tiles, block); };
            while (parts() * k.m * sizeof(float2) > CE_PARTS_BYTES && (size_t)block < tiles) block *= 2;  // more tiles to a unit where there are very many queries
            slots = (int)parts();
            partial = space.take<float2>((size_t)k.m * slots);
            target_scores = space.take<float>(k.m);
            return;
        }
        const size_t lines = tiles_q * TG_M;
        terms = space.take<float>(lines), factors = space.take<float>(lines), own = space.take<float>(k.m);
        cols = space.take<int>(lines);
        if (k.type == CULSH_F16) amax = space.take<uint32_t>(1);
        // G stays on the SM where rows are short enough.  There | by pieces (us): 4,096 x 1M x 128 3,361 | 10,005, x 200,000 x 64 780 | 1,954, x 200,000 x 256 1,410 |
        // 3,101; 500 x 200,000 x 256 286 | 441; but 64 x 200,000 x 128, half the lanes idle, 137 | 111
        const bool fused = k.planes() == 1 && k.d <= 256;
        fused_q = need_q && fused, fused_x = need_x && fused;
        shift = k.type == CULSH_F16 && (fused_q || fused_x) ? CE_HALF_SHIFT : 0;
        if (need_x) {
            sums = space.take<float>((size_t)k.m * k.d);
            // targets of few rows, which many queries share, are summed up for some hundred queries at a time
            own_splits = (int)std::max<size_t>(1, std::min<size_t>({ceil_div(k.m, 512), 16, (size_t)k.c->sm_count / ceil_div(k.n, own_rows(k))}));
            where = space.take<int>((size_t)own_splits * k.n);
        }
        // a unit's tiles of the other side: the last wave full, and four tiles' time for the units' ends; at most 32,768 entries in a sum
        const int nb = k.d > 128 ? 64 : 128;
        auto block_of = [&](size_t own, size_t tiles, size_t most) {
            size_t best = ~(size_t)0;
            int block = 1;
            const size_t least = ceil_div(tiles, 32768 / nb);
            for (size_t blocks = least; blocks <= std::min(tiles, least + most); ++blocks) {
                const size_t per = ceil_div(tiles, blocks), time = ceil_div(own * ceil_div(tiles, per), sms) * (per + 4);
                if (time < best) best = time, block = (int)per;
            }
            return block;
        };
        // split sums grow with both sides: as many queries or rows at a time as CE_PARTS_BYTES hold of
        auto some = [&](int entries, int splits) {
            const size_t fit = CE_PARTS_BYTES / ((size_t)splits * k.d * sizeof(float)) / TG_M * TG_M;
            return (int)std::min<size_t>(entries, std::max<size_t>(fit, TG_M));
        };
        if (fused_q) {
            const size_t tiles = ceil_div(k.n, nb);
            fused_block = block_of(tiles_q, tiles, ceil_div((size_t)4 * sms, tiles_q));
            splits_q = (int)ceil_div(tiles, fused_block), some_q = some(k.m, splits_q);
            acc_q = space.take<float>((size_t)splits_q * some_q * k.d);
        }
        if (fused_x) {  // sums of few rows are split too
            const size_t own = ceil_div(k.n, TG_M), tiles = ceil_div(k.m, nb);
            fused_block_x = own >= (size_t)sms ? (int)ceil_div(tiles, ceil_div(tiles, 32768 / nb)) : block_of(own, tiles, sms / own);
            splits_x = (int)ceil_div(tiles, fused_block_x), some_x = splits_x > 1 ? some(k.n, splits_x) : k.n;
            if (splits_x > 1) parts_x = space.take<float>((size_t)splits_x * some_x * k.d);
        }
        if ((!need_q || fused_q) && (!need_x || fused_x)) return;
        const bool pieces_x = need_x && !fused_x;
        const size_t row_bytes = (size_t)2 * k.planes() * k.m;
        const size_t fit = std::min((k.planes() == 3 ? 4 : 1) * CE_G_BYTES / row_bytes, pieces_x ? CE_PARTS_BYTES / ((size_t)4 * k.d) : ~(size_t)0) / CE_BN * CE_BN;
        // the last wave of the products' units full, with as few pieces as that allows
        const size_t most = std::min(std::max<size_t>(fit / CE_BN, 1), tiles_n), wide = pairs(k.m) ? sms / 2 : sms, high = ceil_div(k.m, pairs(k.m) ? 2 * TG_M : TG_M);
        size_t least_time = ~(size_t)0;
        for (size_t p = most, step = most / 64 + 1; p >= std::max<size_t>(1, most / 3); p -= std::min(p, step)) {
            const size_t rest = tiles_n % p, time = tiles_n / p * (ceil_div(high * p, wide) * 8 + 1) + (rest ? ceil_div(high * rest, wide) * 8 + 1 : 0);
            if (time < least_time) least_time = time, piece = (int)(p * CE_BN);
        }
        G = space.take<uint16_t>((size_t)k.planes() * k.m * piece);
        const int bn = product_bn(k.d);
        const size_t tn = ceil_div(k.d, bn);
        auto split = [&](size_t tiles, int kb, int& splits, int& per) {
            const int most = k.type == CULSH_F32 ? 16 : 512;  // steps of 64 in one accumulator: its adds cut off, 2^-24 of it at a time
            const size_t want = std::max<size_t>(ceil_div(kb, most), std::min<size_t>(sms / std::max<size_t>(tiles, 1), kb / 2));
            per = (int)ceil_div(kb, std::max<size_t>(want, 1));
            splits = (int)ceil_div(kb, per);
        };
        if (need_q && !fused_q) {
            split(tiles_q * tn, (int)ceil_div(std::min(piece, k.n), 64), splits_q, per_q);
            acc_q = space.take<float>((size_t)splits_q * k.m * k.d);
        }
        if (pieces_x) {
            split(ceil_div(std::min(piece, k.n), TG_M) * tn, (int)ceil_div(k.m, 64), splits_x, per_x);
            if (splits_x > 1) parts_x = space.take<float>((size_t)splits_x * piece * k.d);
        }
    }
    static int own_rows(const CeCall& k) { return (int)std::min<size_t>(CE_OWN_ROWS, ceil_div(ceil_div(k.n, 2 * (size_t)k.c->sm_count), 8) * 8); }
    // A pair of CTAs wants 256 entries of the M side; fewer are left to single ones.
    static bool pairs(int64_t rows) { return rows > TG_M; }
    // Of the scores of n rows.
    static CeTile tile_of(const CeCall& k, int64_t n) {
        if (ceil_div(k.m, TG_M) * ceil_div(n, CE_BN) <= (size_t)k.c->sm_count / 4) return CE_SMALL;
        return pairs(k.m) ? CE_PAIR : CE_ONE;
    }
    static int segment_of(const CeCall& k) { return k.m <= 32 || tile_of(k, k.n) == CE_SMALL ? CE_SEGMENT_SMALL : CE_SEGMENT; }
    static int tile_rows(CeTile t) { return t == CE_SMALL ? CE_PART : CE_BN; }
    static int product_bn(int d) { return d > 128 ? 256 : d > 64 ? 128 : 64; }
};

inline unsigned ce_grid(size_t threads) {
    const size_t g = ceil_div(threads, 256);
    if (g > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "the matrices are too large for one call");
    return (unsigned)g;
}

// Planes where they are needed, and where the products find both operands.
struct CeOperands {
    const void *q, *x;
    int64_t ldq, ldx;
    // Also what the gradient needs of the queries, where `a` says where it comes from.
    CeOperands(const CeCall& k, const CePlan& p, CePrepare a) : q(k.Q), x(k.X), ldq(k.ldq), ldx(k.ldx) {
        a.m = k.m, a.n = k.n, a.d = k.d, a.pitch = k.pitch(), a.bias = k.bias, a.bias2 = p.bias2, a.targets = k.targets, a.Q = k.Q, a.ldq = k.ldq;
        uint64_t end = 0;
        auto job = [&](int i, size_t ctas) {
            end += ctas;
            if (end > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "the matrices are too large for one call");
            a.ends[i] = (unsigned)end;
        };
        auto planes = [&](const void* from, int64_t ld, int rows, const float* bias, uint16_t* to) {
            a.planes[to == p.x_planes] = CePlanes{from, ld, rows, bias, to, aligned16(from, ld * (k.type == CULSH_F32 ? 4 : 2))};
            return ceil_div((size_t)rows * k.pitch() / 8, 256);
        };
        job(0, p.q_planes ? planes(k.Q, k.ldq, k.m, nullptr, p.q_planes) : 0);
        job(1, p.x_planes ? planes(k.X, k.ldx, k.n, k.bias, p.x_planes) : 0);
        job(2, p.bias2 ? ceil_div((size_t)k.n + 127, 256) : 0);
        job(3, p.terms ? ceil_div((size_t)k.m + 127, 256) : 0);
        a.terms = p.terms, a.factors = p.factors, a.own = p.own, a.sums = p.sums, a.cols = p.cols, a.where = p.where, a.amax = p.amax;
        a.shift = p.shift, a.t_shift = k.t_shift(), a.lines = p.fused_x;
        // rows, and where they are few and long columns, in shares for some CTAs an SM
        const size_t ctas = 2 * (size_t)k.c->sm_count;
        a.own_rows = CePlan::own_rows(k);
        const size_t tiles = ceil_div(k.n, a.own_rows), shares = std::min(ceil_div(k.d, 32 * CE_OWN_COLS), std::max<size_t>(1, 4 * ctas / tiles));
        a.own_cols = (int)(ceil_div(ceil_div(k.d, shares), 32 * CE_OWN_COLS) * 32 * CE_OWN_COLS);
        a.own_shares = (int)ceil_div(k.d, a.own_cols);
        a.own_tiles = (int)tiles, a.own_queries = (int)ceil_div(k.m, p.own_splits);
        job(4, p.where ? tiles * a.own_shares * p.own_splits : 0);
        if (p.q_planes) q = p.q_planes, ldq = k.pitch();
        if (p.x_planes) x = p.x_planes, ldx = k.pitch();
        if (!end) return;
        if (k.type == CULSH_F32) ce_prepare_kernel<float, 3><<<(unsigned)end, 256, 0, k.stream>>>(a);
        else if (k.type == CULSH_F16) ce_prepare_kernel<__half, 1><<<(unsigned)end, 256, 0, k.stream>>>(a);
        else ce_prepare_kernel<__nv_bfloat16, 1><<<(unsigned)end, 256, 0, k.stream>>>(a);
        KERNEL_CHECK();
    }
    CUtensorMap map_q(const CeCall& k, int box) const { return map_q(k, box, 0, k.m); }
    CUtensorMap map_x(const CeCall& k, int box) const { return map_x(k, box, 0, k.n); }
    // `count` of them from `first` on.
    CUtensorMap map_q(const CeCall& k, int box, int first, int count) const { return map(k, q, ldq, k.m, box, first, count); }
    CUtensorMap map_x(const CeCall& k, int box, int first, int count) const { return map(k, x, ldx, k.n, box, first, count); }
    static CUtensorMap map(const CeCall& k, const void* from, int64_t ld, int rows, int box, int first, int count) {
        return tg_map(static_cast<const uint16_t*>(from) + first * ld, k.tg(), count, k.d, ld, k.planes(), (int64_t)rows * ld * 2, box);
    }
};

// f(number of planes, whether there is a bias, whether K is taken in segments, the tile), as types.
template <typename F>
inline void ce_by(F&& f, bool three, bool bias, bool segments, CeTile tile) {
    auto one = [](bool v, auto&& g) {
        if (v) g(std::true_type());
        else g(std::false_type());
    };
    one(bias, [&](auto b) {
        one(segments, [&](auto s) {
            auto with = [&](auto t) {
                if (three) f(std::integral_constant<int, 3>(), b, s, t);
                else f(std::integral_constant<int, 1>(), b, s, t);
            };
            if (tile == CE_PAIR) with(std::integral_constant<int, CE_PAIR>());
            else if (tile == CE_SMALL) with(std::integral_constant<int, CE_SMALL>());
            else with(std::integral_constant<int, CE_ONE>());
        });
    });
}
inline CeScoreArgs ce_score_args(const CeCall& k, const CePlan& p, CeTile tile, int n0, int n1) {
    CeScoreArgs a{};
    a.d_error = k.d_error, a.idesc = tg_idesc(k.tg(), false, false);
    a.m = k.m, a.kb = (int)ceil_div(k.d, 64), a.segment = CePlan::segment_of(k), a.n0 = n0, a.n1 = n1;
    a.m_tile = tile == CE_PAIR ? 2 * TG_M : TG_M;
    a.tiles_q = (int)ceil_div(k.m, a.m_tile), a.tiles_n = (unsigned)ceil_div(n1 - n0, CePlan::tile_rows(tile));
    a.c = k.c2(), a.bias = p.bias2, a.targets = k.targets;
    return a;
}
inline int ce_box_x(CeTile tile) { return tile == CE_PAIR ? CE_BN / 2 : CePlan::tile_rows(tile); }

inline void cross_entropy(const CeCall& k, float* losses, float* lse, float* lse_low, void* workspace) {
    const CePlan p(k, false, false, false, workspace);
    const CeOperands ops(k, p, CePrepare{});
    CeScoreArgs a = ce_score_args(k, p, p.tile, 0, k.n);
    a.down = k.down(), a.c /= a.down;
    if (p.few) {
        auto go = [&](auto queries) {
            constexpr int M = decltype(queries)::value;
            auto kern = k.bias ? ce_few_kernel<M, true> : ce_few_kernel<M, false>;
            launch_next(k.stream, kern, (size_t)p.slots, (unsigned)CE_FEW_THREADS, 0, static_cast<const float*>(k.Q), k.ldq, static_cast<const float*>(k.X), k.ldx, k.m, k.n, k.d, k.bias,
                        a.c, a.down, k.targets, p.partial, p.target_scores);
            KERNEL_CHECK();
        };
        if (k.m == 1) go(std::integral_constant<int, 1>());
        else if (k.m <= 4) go(std::integral_constant<int, 4>());
        else if (k.m <= 8) go(std::integral_constant<int, 8>());
        else go(std::integral_constant<int, CE_FEW>());
    } else {
    a.block = p.block, a.slots = p.slots, a.partial = p.partial, a.target_scores = p.target_scores;
    const size_t units = ceil_div(a.tiles_n, p.block) * a.tiles_q;
    if (units >= 1ull << 31) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", k.m, k.n);
    a.units = (unsigned)units;
    const CUtensorMap tq = ops.map_q(k, TG_M), tx = ops.map_x(k, ce_box_x(p.tile));
    const bool segments = a.kb > a.segment;
    ce_by([&](auto planes, auto bias, auto segs, auto tile) {
        tc_gemm<CeLossPolicy<decltype(planes)::value, decltype(bias)::value, decltype(segs)::value, decltype(tile)::value>>(k.c, tq, tx, a, k.stream);
    }, k.planes() == 3, k.bias != nullptr, segments, p.tile);
    }
    auto join = p.slots > 256 ? ce_join_kernel<8> : ce_join_kernel<1>;
    launch_next(k.stream, join, ceil_div(k.m, p.slots > 256 ? 1 : 8), 256u, 0, (const float2*)p.partial, p.slots, k.m, k.n, k.targets, p.target_scores, p.bias2, a.c, a.down, losses, lse, lse_low);
    KERNEL_CHECK();
}

// One side of the last launch.
template <typename T>
inline CeFinish ce_finish_of(const CeCall& k, const float* parts, int splits, int64_t rows, const float* factors, const int* which, T* out, int64_t ldo) {
    CeFinish f{};
    f.parts = parts, f.splits = splits, f.split_stride = rows * k.d, f.factors = factors, f.which = which, f.out = out, f.ldo = ldo;
    f.wide = k.d % 4 == 0 && ldo % 4 == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0;
    f.units = rows * (k.d / (f.wide ? 4 : 1));
    f.blocks = ce_grid((size_t)f.units);
    return f;
}
template <typename T>
inline void ce_finish(const CeCall& k, const CePlan& p, const CeFinish& rows, const CeFinish& queries, int q0 = 0) {
    CeFinishArgs a{};
    a.own_splits = p.own_splits, a.where_stride = k.n;
    a.rows = rows, a.queries = queries, a.d = k.d, a.amax = p.amax, a.own = p.own + q0, a.sums = p.sums, a.X = k.X, a.ldx = k.ldx, a.inv_t = k.inv_t();
    const size_t grid = (size_t)rows.blocks + queries.blocks;
    if (!grid) return;
    if (grid > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "the matrices are too large for one call");
    launch_next(k.stream, ce_finish_kernel<T>, grid, 256u, 0, a);
    KERNEL_CHECK();
}

template <int PLANES, bool AMN>
inline void ce_product(const CeCall& k, const CUtensorMap& tg, const void* b, int64_t ldb, int64_t b_rows, CeProductArgs a, int per, int splits) {
    const int bn = CePlan::product_bn(k.d);
    a.d_error = k.d_error, a.idesc = tg_idesc(k.tg(), AMN, true);
    a.cols = k.d, a.kper = per;
    const bool pairs = bn == 256 && CePlan::pairs(a.rows);
    a.m_tile = pairs ? 2 * TG_M : TG_M;
    a.tiles_m = (int)ceil_div(a.rows, a.m_tile), a.tiles_n = (int)ceil_div(k.d, bn);
    splits = (int)std::min<size_t>(splits, ceil_div(a.kb, per));
    a.units = (unsigned)a.tiles_m * a.tiles_n * splits;
    const CUtensorMap tb = tg_map(b, k.tg(), b_rows, k.d, ldb, k.planes(), b_rows * ldb * 2, 64);
    auto go = [&](auto typed) {
        constexpr int TYPED = decltype(typed)::value;
        if (pairs) tc_gemm<CeProductPolicy<PLANES, AMN, 256, true, TYPED>>(k.c, tg, tb, a, k.stream);
        else if (bn == 256) tc_gemm<CeProductPolicy<PLANES, AMN, 256, false, TYPED>>(k.c, tg, tb, a, k.stream);
        else if (bn == 128) tc_gemm<CeProductPolicy<PLANES, AMN, 128, false, TYPED>>(k.c, tg, tb, a, k.stream);
        else tc_gemm<CeProductPolicy<PLANES, AMN, 64, false, TYPED>>(k.c, tg, tb, a, k.stream);
    };
    if constexpr (AMN) {
        if (a.typed) {
            if constexpr (PLANES == 3) go(std::integral_constant<int, 3>());
            else if (k.type == CULSH_F16) go(std::integral_constant<int, 2>());
            else go(std::integral_constant<int, 1>());
            return;
        }
    }
    go(std::integral_constant<int, 0>());
}

// Sums of `count` queries or rows from own0 on.
template <bool ROWS, bool HALF>
inline void ce_fused(const CeCall& k, const CePlan& p, const CeOperands& ops, int own0, int count, void* out, int64_t ld) {
    const int nb = k.d > 128 ? 64 : 128, kb = k.d > 128 ? 4 : k.d > 64 ? 2 : 1;
    CeFusedArgs a{};
    a.d_error = k.d_error;
    constexpr uint32_t M = (uint32_t)(TG_M >> 4) << 24;
    a.idesc_s = tg_idesc(k.tg(), false, false) | M | ((uint32_t)(nb >> 3) << 17);
    a.idesc_o = tg_idesc(k.tg(), false, true) | M | ((uint32_t)(kb * 64 >> 3) << 17);
    a.own = count, a.other = ROWS ? k.m : k.n, a.own0 = own0;
    a.tiles_own = (int)ceil_div(a.own, TG_M), a.tiles_other = (int)ceil_div(a.other, nb), a.block = ROWS ? p.fused_block_x : p.fused_block;
    const size_t units = ceil_div(a.tiles_other, a.block) * a.tiles_own;
    if (units >= 1ull << 31) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", k.m, k.n);
    a.units = (unsigned)units;
    const int q0 = ROWS ? 0 : own0;
    a.d = k.d, a.c = k.c2(), a.bias = ROWS && p.bias2 ? p.bias2 + own0 : p.bias2, a.terms = p.terms + q0, a.factors = p.factors + q0, a.amax = p.amax, a.target_cols = p.cols + q0;
    a.parts = !ROWS ? p.acc_q : p.splits_x > 1 ? p.parts_x : nullptr, a.out = out, a.ld = ld, a.where = p.where + own0, a.where_stride = k.n, a.own_splits = p.own_splits, a.sums = p.sums, a.inv_t = k.inv_t();
    const CUtensorMap own = ROWS ? ops.map_x(k, TG_M, own0, count) : ops.map_q(k, TG_M, own0, count), other = ROWS ? ops.map_q(k, nb) : ops.map_x(k, nb);
    auto go = [&](auto boxes) {
        constexpr int KB = decltype(boxes)::value;
        if (k.bias) ce_fused_launch<KB, ROWS, true, HALF>(k.c, own, other, a, k.stream);
        else ce_fused_launch<KB, ROWS, false, HALF>(k.c, own, other, a, k.stream);
    };
    if (kb == 4) go(std::integral_constant<int, 4>());
    else if (kb == 2) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 1>());
}

template <typename T>
inline void cross_entropy_backward(const CeCall& k, const float* losses, const float* lse, const float* lse_low, const float* grad_losses, const float* grad_lse, T* grad_Q,
                                   int64_t ld_gq, T* grad_X, int64_t ld_gx, void* workspace) {
    constexpr int PLANES = std::is_same<T, float>::value ? 3 : 1;
    constexpr bool HALF = std::is_same<T, __half>::value;
    const CePlan p(k, true, grad_Q != nullptr, grad_X != nullptr, workspace);
    if (p.amax) CU_CHECK(cudaMemsetAsync(p.amax, 0, 4, k.stream));
    CePrepare before{};
    before.losses = losses, before.lse = lse, before.lse_low = lse_low, before.grad_losses = grad_losses, before.grad_lse = grad_lse;
    const CeOperands ops(k, p, before);
    if constexpr (PLANES == 3) {
        if (p.few) {
            auto go = [&](auto queries) {
                constexpr int M = decltype(queries)::value;
                auto kern = k.bias ? ce_few_grad_kernel<T, M, true> : ce_few_grad_kernel<T, M, false>;
                static thread_local uint64_t ready[2] = {};  // devices whose limit is set
                uint64_t& is = ready[k.bias != nullptr];
                if (k.c->device >= 64 || !(is >> k.c->device & 1)) {
                    CU_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, CE_FEW * CE_FEW_GRAD * 4));
                    if (k.c->device < 64) is |= 1ull << k.c->device;
                }
                launch_next(k.stream, kern, (size_t)p.splits_q, (unsigned)CE_FEW_THREADS, grad_Q ? (size_t)k.m * k.d * 4 : 0, static_cast<const T*>(k.Q), k.ldq, static_cast<const T*>(k.X), k.ldx,
                            k.m, k.n, k.d, k.bias, k.c2(), k.inv_t(), p.terms, p.factors, p.own, p.cols, p.acc_q, grad_X, ld_gx);
                KERNEL_CHECK();
            };
            if (k.m <= 4) go(std::integral_constant<int, 4>());
            else go(std::integral_constant<int, CE_FEW>());
            if (grad_Q) ce_finish<T>(k, p, CeFinish{}, ce_finish_of(k, p.acc_q, p.splits_q, k.m, nullptr, nullptr, grad_Q, ld_gq));
            return;
        }
    }
    CeFinish last{};  // of dX, for the launch that finishes dQ
    int first_q = 0;  // of the queries that it finishes
    if constexpr (PLANES == 1) {
        for (int64_t x0 = 0; p.fused_x && x0 < k.n; x0 += p.some_x) {
            const int here = (int)std::min<int64_t>(p.some_x, k.n - x0);
            ce_fused<true, HALF>(k, p, ops, (int)x0, here, grad_X + x0 * ld_gx, ld_gx);
            if (p.splits_x == 1) continue;
            last = ce_finish_of(k, p.parts_x, p.splits_x, here, nullptr, p.where + x0, grad_X + x0 * ld_gx, ld_gx);
            if (x0 + here < k.n) ce_finish<T>(k, p, last, CeFinish{}), last = CeFinish{};
        }
        for (int64_t q0 = 0; p.fused_q && q0 < k.m; q0 += p.some_q) {
            const int here = (int)std::min<int64_t>(p.some_q, k.m - q0);
            ce_fused<false, HALF>(k, p, ops, (int)q0, here, nullptr, 0);
            first_q = (int)q0;
            if (q0 + here < k.m) {
                ce_finish<T>(k, p, last, ce_finish_of(k, p.acc_q, p.splits_q, here, p.factors + q0, p.cols + q0, grad_Q + q0 * ld_gq, ld_gq), first_q);
                last = CeFinish{};
            }
        }
    }
    const bool pieces_q = grad_Q && !p.fused_q, pieces_x = grad_X && !p.fused_x;
    const CUtensorMap tq = ops.map_q(k, TG_M);
    const int64_t g_plane = (int64_t)k.m * p.piece;
    for (int64_t n0 = 0; (pieces_q || pieces_x) && n0 < k.n; n0 += p.piece) {
        const int here = (int)std::min<int64_t>(p.piece, k.n - n0);
        const CeTile tile = CePlan::tile_of(k, here);
        CeScoreArgs s = ce_score_args(k, p, tile, (int)n0, (int)(n0 + here));
        s.terms = p.terms, s.factors = p.factors, s.shift = p.shift, s.amax = p.amax, s.target_cols = p.cols, s.G = p.G, s.pitch = p.piece, s.plane = g_plane;
        s.block = 1;
        const size_t units = (size_t)s.tiles_n * s.tiles_q;
        if (units >= 1ull << 31) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", k.m, k.n);
        s.units = (unsigned)units;
        const CUtensorMap tx = ops.map_x(k, ce_box_x(tile));
        ce_by([&](auto planes, auto bias, auto segs, auto type) {
            if constexpr (decltype(planes)::value == PLANES)
                tc_gemm<CeGradPolicy<PLANES, decltype(bias)::value, HALF, decltype(segs)::value, decltype(type)::value>>(k.c, tq, tx, s, k.stream);
        }, PLANES == 3, k.bias != nullptr, s.kb > s.segment, tile);
        const int64_t g_cols = (int64_t)s.tiles_n * CePlan::tile_rows(tile);  // behind the last row G has zeros
        if (pieces_x) {
            CeProductArgs a{};
            a.rows = here, a.b0 = 0, a.kb = (int)ceil_div(k.m, 64), a.out = p.parts_x;
            if (p.splits_x == 1) {
                a.typed = grad_X + n0 * ld_gx, a.ld = ld_gx, a.amax = p.amax, a.where = p.where + n0, a.sums = p.sums;
                a.own_splits = p.own_splits, a.where_stride = k.n;
                a.inv_t = k.inv_t();
            }
            ce_product<PLANES, true>(k, tg_map(p.G, k.tg(), k.m, g_cols, p.piece, PLANES, g_plane * 2, 64), ops.q, ops.ldq, k.m, a, p.per_x, p.splits_x);
            if (p.splits_x > 1) {
                last = ce_finish_of(k, p.parts_x, p.splits_x, here, nullptr, p.where + n0, grad_X + n0 * ld_gx, ld_gx);
                if (n0 + here < k.n) ce_finish<T>(k, p, last, CeFinish{}), last = CeFinish{};
            }
        }
        if (pieces_q) {
            CeProductArgs a{};
            a.rows = k.m, a.b0 = (int)n0, a.kb = (int)ceil_div(here, 64), a.out = p.acc_q, a.accumulate = n0 > 0;
            ce_product<PLANES, false>(k, tg_map(p.G, k.tg(), k.m, g_cols, p.piece, PLANES, g_plane * 2, TG_M), ops.x, ops.ldx, k.n, a, p.per_q, p.splits_q);
        }
    }
    CeFinish queries{};
    if (grad_Q) queries = ce_finish_of(k, p.acc_q, p.splits_q, k.m - first_q, p.fused_q ? p.factors + first_q : nullptr, p.cols + first_q, grad_Q + first_q * ld_gq, ld_gq);
    ce_finish<T>(k, p, last, queries, first_q);
}

}  // namespace culsh_b200
