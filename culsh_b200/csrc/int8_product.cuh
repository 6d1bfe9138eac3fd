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
// Products of two scales, squares of one and sums by them are floats where scales are from 2^-62 to 2^46 (a row of zeros may have any): 2^-124 to 2^123.  Elsewhere they may leave the range that the
// score itself is in, and are taken in parts.
__device__ __forceinline__ bool i8_far(int metric, float scale, int squares) {
    return metric != MX_COSINE && squares != 0 && __float_as_uint(scale) - __float_as_uint(0x1p-62f) >= __float_as_uint(0x1p46f) - __float_as_uint(0x1p-62f);  // as floats are in their bits' order
}
__device__ __forceinline__ int i8_exponent(float scale) { return (__float_as_int(scale) >> 23 & 255) - 127; }
__device__ __forceinline__ float i8_power(int e) { return __int_as_float((e + 127) << 23); }
// Each scale as two of half its exponent; distances by scales over the larger one's power of two.
__device__ __forceinline__ float i8_score_far(int metric, int dot, float q_scale, float q_squares, float x_scale, float x_squares) {
    const int eq = i8_exponent(q_scale), ex = i8_exponent(x_scale);
    if (metric == MX_EUCLIDEAN) {
        const int e = min(max(eq, ex), 126);
        const float q = q_scale * i8_power(-e), x = x_scale * i8_power(-e);
        return (fmaf(2.f, (float)dot * (q * x), -(q_squares * (q * q))) - x_squares * (x * x)) * i8_power(e) * i8_power(e);
    }
    const int hq = eq >> 1, hx = ex >> 1;
    return (float)dot * (q_scale * i8_power(-hq) * (x_scale * i8_power(-hx))) * (i8_power(hq) * i8_power(hx));
}

struct I8ProductArgs {
    int* d_error;
    unsigned block_units;     // of a block of tiles, all chunks
    unsigned units, step;     // units between one of a CTA, or of a pair, and its next
    uint32_t idesc;
    int n, nq, kb, metric, chunks, block;
    unsigned tiles;
    const float *scales, *q_scales;
    const int32_t *squares, *q_squares;
    void* out;
    int64_t ld;
    bool wide, small;         // rows of the result begin at multiples of 16 bytes; sums are below 2^22
};
constexpr int I8_FEW = 64, I8_FEWEST = 16, I8_SHORT = 2;  // queries; steps of K of short rows
struct I8Unit {
    static constexpr int tiles = 1, k0 = 0;
    unsigned u;
    int tile, chunk, k1;
    __device__ __forceinline__ I8Unit(const I8ProductArgs& a, unsigned u_) : u(u_) {  // blocks of neighbouring tiles, a chunk of the queries after the other in each
        const unsigned b = u / a.block_units, left = u - b * a.block_units;
        const unsigned here = min((unsigned)a.block, a.tiles - b * (unsigned)a.block);
        chunk = (int)(left / here);
        tile = (int)(b * (unsigned)a.block + (left - (unsigned)chunk * here));
        k1 = a.kb;
    }
};
// A scale and squares on their way.
struct I8Fetch {
    float scale = 0.f;
    int squares = 0;
    __device__ __forceinline__ void get(const float* scales, const int32_t* from, int at, int end) {
        const bool in = at < end;
        scale = in ? __ldcg(scales + at) : 0.f;
        squares = in ? __ldcg(from + at) : 0;
    }
    __device__ __forceinline__ bool far(int metric) const { return i8_far(metric, scale, squares); }
    // What a score takes, and a far one.
    __device__ __forceinline__ float2 terms(int metric) const { return i8_terms(metric, scale, squares); }
    __device__ __forceinline__ float2 far_terms() const { return make_float2(scale, (float)squares); }
};
__device__ __forceinline__ float i8_score(int metric, int dot, const I8Fetch& q, const I8Fetch& x) {
    if (q.far(metric) || x.far(metric)) return i8_score_far(metric, dot, q.scale, (float)q.squares, x.scale, (float)x.squares);
    const float2 qt = q.terms(metric), xt = x.terms(metric);
    const float v = (float)dot * (qt.x * xt.x);
    return metric == MX_EUCLIDEAN ? fmaf(2.f, v, -qt.y) - xt.y : v;
}
// The scores of N sums; conversions of whole numbers run at an eighth of the rate of additions, which do the same for what fits the fraction of a float.
template <int N>
__device__ __forceinline__ void i8_scores(int metric, bool small, uint32_t (&r)[N], float2 q, const float* factors, const float* terms) {
    const uint64_t qq = f2_pack(q.x, q.x);
    auto all = [&](auto convert) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(factors + j);
            float v[4];
            f2_unpack(f2_mul(convert(r[j], r[j + 1]), f2_mul(qq, x.x)), v[0], v[1]);
            f2_unpack(f2_mul(convert(r[j + 2], r[j + 3]), f2_mul(qq, x.y)), v[2], v[3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) r[j + k] = __float_as_uint(v[k]);
        }
    };
    if (small) {
        const uint64_t minus = f2_pack(-12582912.f, -12582912.f);  // 1.5 x 2^23
        all([&](uint32_t lo, uint32_t hi) { return f2_add(f2_pack(__uint_as_float(0x4B400000u + lo), __uint_as_float(0x4B400000u + hi)), minus); });
    } else {
        all([](uint32_t lo, uint32_t hi) { return f2_pack((float)(int)lo, (float)(int)hi); });
    }
    if (metric == MX_EUCLIDEAN) {
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = __float_as_uint(fmaf(2.f, __uint_as_float(r[j]), -q.y) - terms[j]);
    }
}

// A lane's `columns` scores of a tile with far ones, the first `left` of them stored `step` entries apart.  Seldom taken, and apart: in the loop of the others its registers made
// 1,000 x 1M x 128 take 642 to 770 us in place of 623.
template <typename OUT>
__device__ __noinline__ void i8_store_far(int metric, uint32_t taddr, int columns, int left, float2 mine, const float* factors, const float* squares, OUT* out, int64_t step) {
#pragma unroll 1
    for (int c0 = 0; c0 < columns; c0 += 16) {
        uint32_t r[16];
        tg_ld16(taddr + c0, r);
        tc_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (c0 + j < left) store_score(out + (c0 + j) * step, i8_score_far(metric, (int)r[j], mine.x, mine.y, factors[c0 + j], squares[c0 + j]));
    }
    __syncwarp();
}

// More than 64 queries: they are the M side, a lane of the accumulator a query.  Short rows leave the time to the epilogue: a warp has 32 queries by all 128 rows of a tile, and groups of four
// take tiles in turn; of long rows a tile has 256, and a warp 64 of them.  128 bytes of each query are stored at a time, by way of shared memory.  4,099 x 32,771 x 2,048 265 us, the tensor pipe
// busy for 68 % (one CTA by 128 rows 414); 1,000 x 1M x 128 bfloat16 619 to 640, no unit above 38 % (conversions in place of additions 923).
template <typename OUT, bool PAIRS, int N>
struct I8ProductPolicy {
    static constexpr bool A_MN = false, B_MN = false, I8 = true, PARTS = N == 256, PAIR = PAIRS;
    static constexpr int BN = N, EPI_WARPS = 16, PART = PARTS ? BN / 4 : BN, TURNS = PARTS ? 1 : EPI_WARPS / 4, SEGMENTS = 0, PIECE = 32 * 128, EPI_BYTES = EPI_WARPS * (PIECE + PART * 8);
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
        float *factors, *terms;
        I8Fetch row[PART / 32], query;
        __device__ __forceinline__ Epilogue(const Args& a, unsigned char* smem, int warp, int quarter_, int group_, int lane_, int rank_)
            : quarter(quarter_), group(group_), lane(lane_), rank(rank_), piece(smem + warp * PIECE),
              factors(reinterpret_cast<float*>(smem + EPI_WARPS * PIECE) + warp * 2 * PART), terms(factors + PART) {
            const unsigned first = (PAIR ? blockIdx.x >> 1 : blockIdx.x) + (PARTS ? 0u : group * a.step);
            if (first < a.units) fetch(a, Unit(a, first));
        }
        __device__ __forceinline__ int first_query(const Unit& u) const { return u.chunk * (PAIR ? 2 * TG_M : TG_M) + rank * TG_M + quarter * 32; }
        __device__ __forceinline__ int first_row(const Unit& u) const { return u.tile * BN + (PARTS ? group * PART : 0); }
        __device__ __forceinline__ void fetch(const Args& a, const Unit& u) {
            query.get(a.q_scales, a.q_squares, first_query(u) + lane, a.nq);
#pragma unroll
            for (int i = 0; i < PART / 32; ++i) row[i].get(a.scales, a.squares, first_row(u) + i * 32 + lane, a.n);
        }
        __device__ __forceinline__ void unit_begin(const Args&, const Unit&) {}
        __device__ __forceinline__ void unit_end(const Args&, const Unit&) {}
        template <typename D>
        __device__ __forceinline__ void tile(const Args& a, const Unit& u, int, uint32_t taddr, bool live, bool, D&& done) {
            constexpr int PER = 128 / sizeof(OUT), V = 16 / sizeof(OUT);  // scores of a query in a piece, in a store
            const int q0 = first_query(u), n0 = first_row(u);
            float2 mine = query.terms(a.metric);
            bool far = query.far(a.metric);
#pragma unroll
            for (int i = 0; i < PART / 32; ++i) {
                const float2 x = row[i].terms(a.metric);
                factors[i * 32 + lane] = x.x, terms[i * 32 + lane] = x.y;
                far = far || row[i].far(a.metric);
            }
            far = __any_sync(0xFFFFFFFFu, far);
            if (far) {
                mine = query.far_terms();
#pragma unroll
                for (int i = 0; i < PART / 32; ++i) {
                    const float2 x = row[i].far_terms();
                    factors[i * 32 + lane] = x.x, terms[i * 32 + lane] = x.y;
                }
            }
            if (!live) mine.x = __int_as_float(0x7FFFFFFF);
            __syncwarp();
            if (a.units - u.u > TURNS * a.step) fetch(a, Unit(a, u.u + TURNS * a.step));  // on its way while this unit is worked on
            if (q0 >= a.nq || n0 >= a.n) {
                done();
                return;
            }
            OUT* const o = reinterpret_cast<OUT*>(a.out) + (int64_t)q0 * a.ld + n0;
            if (far) {
                i8_store_far(a.metric, taddr, PART, q0 + lane < a.nq ? a.n - n0 : 0, mine, factors, terms, o + lane * a.ld, 1);
                done();
                return;
            }
#pragma unroll 1
            for (int p0 = 0; p0 < PART; p0 += PER) {
#pragma unroll
                for (int c0 = 0; c0 < PER; c0 += 32) {
                    uint32_t r[32];
                    tg_ld32(taddr + p0 + c0, r);
                    tc_ld_wait();
                    if (p0 + c0 + 32 == PART) done();
                    i8_scores(a.metric, a.small, r, mine, factors + p0 + c0, terms + p0 + c0);
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
                        *reinterpret_cast<uint4*>(piece + lane * 128 + (((c0 / V + i) ^ (lane & 7)) << 4)) = w;
                    }
                }
                __syncwarp();
                const int rows = a.nq - q0, left = a.n - n0 - p0;
                if (a.wide && rows >= 32 && left >= PER) {  // eight lanes a row
                    OUT* to = o + p0 + (lane >> 3) * a.ld + (lane & 7) * V;
                    uint4 w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int line = i * 4 + (lane >> 3);
                        w[i] = *reinterpret_cast<const uint4*>(piece + line * 128 + (((lane & 7) ^ (line & 7)) << 4));
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i, to += 4 * a.ld) *reinterpret_cast<uint4*>(to) = w[i];
                } else {
#pragma unroll 4
                    for (int i = 0; i < min(rows, 32); ++i) {
#pragma unroll
                        for (int j = lane; j < PER; j += 32) {
                            const OUT* const from = reinterpret_cast<const OUT*>(piece + i * 128 + (((j / V) ^ (i & 7)) << 4)) + j % V;
                            if (j < left) o[i * a.ld + p0 + j] = *from;
                        }
                    }
                }
                __syncwarp();
            }
        }
    };
};

// Up to 64 queries: the rows are the M side, so that no lane is idle, and a warp's store of a query is 32 neighbouring scores.  One query by 1M x 128 36 us, HBM 47 % (151 with the query
// there).  Through the Python calls, here | with the queries there: 17 of them 49 | 100, 48 71 | 95, but 64 85 | 77; by 20,000 x 1,000 17 24.4 | 25.4, 64 24.5 | 18.3.
template <typename OUT, int N>
struct I8FewPolicy {
    static constexpr bool A_MN = false, B_MN = false, I8 = true, PARTS = false, PAIR = false;
    static constexpr int BN = N, EPI_WARPS = 8, SEGMENTS = 0, EPI_BYTES = 1024;
    using Pairs = PlanePairs<1>;
    using Args = I8ProductArgs;
    struct Unit {
        static constexpr int tiles = 1, k0 = 0;
        unsigned u;
        int k1;
        __device__ __forceinline__ Unit(const Args& a, unsigned u_) : u(u_), k1(a.kb) {}
    };
    static __device__ __forceinline__ void load(const Args&, const Unit& u, int, int, int, int k, const CUtensorMap* ta, const CUtensorMap* tb, unsigned char* sa, unsigned char* sb,
                                                uint32_t bar, int) {
        tma_load_3d<false>(sa, ta, bar, k * 128, (int)u.u * TG_M, 0);
        tma_load_3d<false>(sb, tb, bar, k * 128, 0, 0);
    }
    static __device__ __forceinline__ int n_mma(const Args& a, const Unit&, int) { return (a.nq + 15) & ~15; }
    struct Epilogue {
        int quarter, group, lane;
        float *factors, *terms, *squares;  // of the queries, the same for all warps
        bool far = false;                  // one of them is
        I8Fetch row;
        __device__ __forceinline__ Epilogue(const Args& a, unsigned char* smem, int, int quarter_, int group_, int lane_, int)
            : quarter(quarter_), group(group_), lane(lane_), factors(reinterpret_cast<float*>(smem)), terms(factors + I8_FEW), squares(terms + I8_FEW) {
#pragma unroll
            for (int i = lane; i < I8_FEW; i += 32) {
                I8Fetch f;
                f.get(a.q_scales, a.q_squares, i, a.nq);
                const float2 q = i8_terms(a.metric, f.scale, f.squares);
                factors[i] = q.x, terms[i] = q.y, squares[i] = (float)f.squares;
                far = far || f.far(a.metric);
            }
            far = __any_sync(0xFFFFFFFFu, far);
            // the groups take the CTA's units in turn
            const unsigned first = blockIdx.x + group * a.step;
            if (first < a.units) row.get(a.scales, a.squares, (int)first * TG_M + quarter * 32 + lane, a.n);
        }
        __device__ __forceinline__ void unit_begin(const Args&, const Unit&) {}
        __device__ __forceinline__ void unit_end(const Args&, const Unit&) {}
        template <typename D>
        __device__ __forceinline__ void tile(const Args& a, const Unit& u, int, uint32_t taddr, bool live, bool, D&& done) {
            const int at = (int)u.u * TG_M + quarter * 32 + lane;
            const bool some_far = far || __any_sync(0xFFFFFFFFu, row.far(a.metric));
            float2 mine = some_far ? row.far_terms() : row.terms(a.metric);
            if (!live) mine.x = __int_as_float(0x7FFFFFFF);
            const uint64_t next = (uint64_t)u.u + 2ull * a.step;
            if (next < a.units) row.get(a.scales, a.squares, (int)next * TG_M + quarter * 32 + lane, a.n);
            OUT* o = reinterpret_cast<OUT*>(a.out) + at;
            if (some_far) {
                i8_store_far(a.metric, taddr, a.nq, at < a.n ? a.nq : 0, mine, factors, squares, o, a.ld);
                done();
                return;
            }
#pragma unroll 1
            for (int q0 = 0; q0 < a.nq; q0 += 16) {
                uint32_t r[16];
                tg_ld16(taddr + q0, r);
                tc_ld_wait();
                if (q0 + 16 >= a.nq) done();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (at >= a.n || q0 + j >= a.nq) break;
                    const float v = (float)(int)r[j] * (factors[q0 + j] * mine.x);
                    store_score(o, a.metric == MX_EUCLIDEAN ? fmaf(2.f, v, -terms[q0 + j]) - mine.y : v);
                    o += a.ld;
                }
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
    int64_t share;            // candidates of a warp
    int n, nq, pitch, metric;
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
// A warp takes its share of the candidates, 32 at a time; LANES threads one of them, 16 bytes of its row each (and every 16 LANES of a longer one), with up to eight rows' loads in flight.
// The list that a candidate belongs to is searched for once, and again where it ends.  Bound by the gathers: 15M candidates of 1M x 128 by cosine 530 us; with a search for each candidate's list and one row at a time 990.
template <int LANES>
__global__ void __launch_bounds__(256) i8_score_kernel(I8ScoreArgs a, KernelBefore before) {
    behind_kernel_before(before);
    constexpr int GROUPS = 32 / LANES, AHEAD = LANES < 8 ? LANES : 8;
    const int lane = threadIdx.x & 31, at = lane % LANES, group = lane / LANES;
    const int64_t warp = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), first = warp * a.share, last = min(first + a.share, a.total);
    if (first >= last) return;
    int list = i8_owner(a.offsets, 0, a.nq, first);
    int64_t end = __ldcg(a.offsets + list + 1);
    const int64_t column = (int64_t)at * 16;
    const bool one = a.pitch <= LANES * 16, mine_in = column < a.pitch;
    uint4 held = make_uint4(0u, 0u, 0u, 0u);  // of the query that is worked on
    int held_list = -1;
    for (int64_t c0 = first; c0 < last; c0 += 32) {
        const int64_t c = c0 + lane, to = min(c0 + 31, last - 1);
        const bool in = c < last;
        const int id = in ? __ldcg(a.ids + c) : -1;
        const bool real = (unsigned)id < (unsigned)a.n;
        // a sector each: only what the metric takes
        const float scale = real && a.metric != MX_COSINE ? __ldcg(a.scales + id) : 0.f;
        const int squares = real && a.metric != MX_DOT ? __ldcg(a.squares + id) : 0;
        int owner = list;
        const bool same = to < end;  // for the whole warp
        if (!same) {
            owner = i8_owner(a.offsets, list, a.nq, in ? c : to);
            list = __shfl_sync(0xFFFFFFFFu, owner, 31);
            end = __ldcg(a.offsets + list + 1);
        }
        if (same && one && held_list != list) {
            if (mine_in) held = __ldcg(reinterpret_cast<const uint4*>(a.q_codes + (int64_t)list * a.pitch + column));
            held_list = list;
        }
        I8Fetch q, x;
        q.scale = __ldcg(a.q_scales + owner), q.squares = __ldcg(a.q_squares + owner);
        x.scale = scale, x.squares = a.metric == MX_DOT ? 1 : squares;  // as if no row were zeros
        int mine = 0;
#pragma unroll 1
        for (int i0 = 0; i0 < LANES; i0 += AHEAD) {
            int dot[AHEAD];
            if (one) {
                uint4 v[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int row = __shfl_sync(0xFFFFFFFFu, id, (i0 + i) * GROUPS + group);
                    v[i] = make_uint4(0u, 0u, 0u, 0u);
                    if ((unsigned)row < (unsigned)a.n && mine_in) v[i] = __ldcg(reinterpret_cast<const uint4*>(a.codes + (int64_t)row * a.pitch + column));
                }
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    uint4 w = held;
                    if (!same) {
                        const int from = __shfl_sync(0xFFFFFFFFu, owner, (i0 + i) * GROUPS + group);
                        if (mine_in) w = __ldcg(reinterpret_cast<const uint4*>(a.q_codes + (int64_t)from * a.pitch + column));
                    }
                    dot[i] = __dp4a((int)v[i].w, (int)w.w, __dp4a((int)v[i].z, (int)w.z, __dp4a((int)v[i].y, (int)w.y, __dp4a((int)v[i].x, (int)w.x, 0))));
                }
            } else {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int row = __shfl_sync(0xFFFFFFFFu, id, (i0 + i) * GROUPS + group), from = __shfl_sync(0xFFFFFFFFu, owner, (i0 + i) * GROUPS + group);
                    dot[i] = 0;
                    if ((unsigned)row < (unsigned)a.n) {
                        const int8_t *const rows = a.codes + (int64_t)row * a.pitch, *const queries = a.q_codes + (int64_t)from * a.pitch;
#pragma unroll 4
                        for (int k = (int)column; k < a.pitch; k += LANES * 16) {
                            const uint4 v = __ldcg(reinterpret_cast<const uint4*>(rows + k)), w = __ldcg(reinterpret_cast<const uint4*>(queries + k));
                            dot[i] = __dp4a((int)v.w, (int)w.w, __dp4a((int)v.z, (int)w.z, __dp4a((int)v.y, (int)w.y, __dp4a((int)v.x, (int)w.x, dot[i]))));
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
                for (int o = 1; o < LANES; o *= 2) dot[i] += __shfl_xor_sync(0xFFFFFFFFu, dot[i], o);
                const int sum = __shfl_sync(0xFFFFFFFFu, dot[i], (lane % GROUPS) * LANES);
                if (lane / GROUPS == i0 + i) mine = sum;
            }
        }
        if (in) a.out[c] = real ? i8_score(a.metric, mine, q, x) : __int_as_float(0x7FFFFFFF);
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
    const int pitch = i8_pitch(d);
    const bool few = nq <= I8_FEW, pairs = nq > TG_M;
    const bool brief = a.kb <= I8_SHORT;
    const int side = few || brief ? 128 : 256;  // rows of a tile
    a.chunks = few ? 1 : (int)ceil_div(nq, pairs ? 2 * TG_M : TG_M), a.tiles = (unsigned)ceil_div(n, side), a.block = c->sm_count / 2;
    if ((uint64_t)a.tiles * a.chunks >= (1ull << 31)) fail(CULSH_ERR_UNSUPPORTED, "%d queries by %d rows are too many for one call", nq, n);
    a.units = a.tiles * (unsigned)a.chunks;
    a.step = std::min<unsigned>(a.units, (unsigned)(pairs ? c->sm_count / 2 : c->sm_count));
    a.block_units = (unsigned)std::min<uint64_t>((uint64_t)a.block * a.chunks, 1ull << 31);
    a.scales = scales, a.q_scales = q_scales, a.squares = squares, a.q_squares = q_squares, a.out = out, a.ld = ld;
    a.wide = aligned16(out, ld * (int64_t)sizeof(OUT));
    a.small = (int64_t)pitch * 127 * 127 < 1 << 22;
    const int box_q = few ? (nq <= I8_FEWEST ? I8_FEWEST : I8_FEW) : TG_M, box_x = few ? TG_M : pairs ? side / 2 : side;
    const CUtensorMap tq = tg_map(q_codes, TG_I8, nq, pitch, pitch, 1, 0, box_q), tx = tg_map(codes, TG_I8, n, pitch, pitch, 1, 0, box_x);
    if (nq <= I8_FEWEST) tc_gemm<I8FewPolicy<OUT, I8_FEWEST>>(c, tx, tq, a, stream);
    else if (few) tc_gemm<I8FewPolicy<OUT, I8_FEW>>(c, tx, tq, a, stream);
    else if (pairs && brief) tc_gemm<I8ProductPolicy<OUT, true, 128>>(c, tq, tx, a, stream);
    else if (pairs) tc_gemm<I8ProductPolicy<OUT, true, 256>>(c, tq, tx, a, stream);
    else if (brief) tc_gemm<I8ProductPolicy<OUT, false, 128>>(c, tq, tx, a, stream);
    else tc_gemm<I8ProductPolicy<OUT, false, 256>>(c, tq, tx, a, stream);
}

inline void i8_score_lists(const CtxPtr& c, I8ScoreArgs a, cudaStream_t stream) {
    const int64_t spans = (int64_t)ceil_div(a.total, 32), most = (int64_t)c->sm_count * 8 * 6;  // warps at a time
    a.share = 32 * (int64_t)ceil_div(spans, std::min<int64_t>(spans, 4 * most));
    const size_t grid = ceil_div(ceil_div(a.total, a.share), 8);
    if (a.pitch <= 16) launch_next(stream, i8_score_kernel<1>, grid, 256u, 0, a);
    else if (a.pitch <= 32) launch_next(stream, i8_score_kernel<2>, grid, 256u, 0, a);
    else if (a.pitch <= 64) launch_next(stream, i8_score_kernel<4>, grid, 256u, 0, a);
    else if (a.pitch <= 128) launch_next(stream, i8_score_kernel<8>, grid, 256u, 0, a);
    else if (a.pitch <= 256) launch_next(stream, i8_score_kernel<16>, grid, 256u, 0, a);
    else launch_next(stream, i8_score_kernel<32>, grid, 256u, 0, a);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
