// Scores of candidate lists: for every (query, candidate) pair of a CSR result the product of the query as it is with the row in microscaled 4-bit floating
// point (mx_rows.cuh), or the cosine, or the negative squared distance.  out[c] = sum_k q_k x^[id(c)]_k.
#pragma once

#include "mx_product.cuh"

namespace culsh_b200 {

// Largest i with offsets[i] <= at, i < n, by a warp: 32 of what is left are looked at at a time.
__device__ __forceinline__ int owner_of(const int64_t* __restrict__ offsets, int n, int64_t at) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;  // offsets[lo] <= at < offsets[hi]
    while (hi - lo > 1) {
        const int step = (int)(((unsigned)(hi - lo) + 31u) / 32u);
        const int64_t p = (int64_t)lo + (int64_t)lane * step;
        const unsigned below = __ballot_sync(0xFFFFFFFFu, lane == 0 || (p < hi && __ldg(offsets + p) <= at));
        lo += (31 - __clz((int)below)) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// Scores whose sums pass float32 are NaN, as are those of queries that are not finite: the two kernels below add in different orders, in which infinities of both signs can meet.
__device__ __forceinline__ float finite_or_nan(float v) { return fabsf(v) < INFINITY ? v : __int_as_float(0x7FFFFFFF); }

struct MxScoreArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* norms;
    const int32_t* ids;
    const int64_t* offsets;
    float* out;
    int64_t ldq, total;
    int n, nq, d, groups, metric;
};

// A warp takes `per` neighbouring candidates, eight at a time; four lanes share one and take its blocks of 32 values (16 bytes) in turn.
template <typename T>
__global__ void __launch_bounds__(256) mx_score_kernel(const T* __restrict__ Q, MxScoreArgs a, int per) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    int64_t at = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * per;
    const int64_t end = min(at + per, a.total);
    if (at >= end) return;
    int q = owner_of(a.offsets, a.nq, at);
    while (at < end) {
        int64_t last = __ldg(a.offsets + q + 1);
        if (last <= at) {  // empty, or done
            if (++q == a.nq) return;
            continue;
        }
        last = min(last, end);
        const T* __restrict__ x = Q + (int64_t)q * a.ldq;
        float q2 = 0.f;
        if (a.metric != MX_DOT) {
            bool zero = true;
            for (int i = lane; i < a.d; i += 32) {
                const float v = (float)x[i];
                q2 = fmaf(v, v, q2);
                zero = zero && v == 0.f;
            }
            for (int o = 16; o; o >>= 1) q2 += __shfl_xor_sync(0xFFFFFFFFu, q2, o);
            if (!__all_sync(0xFFFFFFFFu, zero) && q2 == 0.f) q2 = MX_LEAST;
        }
        for (; at < last; at += 8) {
            const int64_t c = at + (lane >> 2);
            const int32_t id = c < last ? __ldg(a.ids + c) : -1;
            const bool ok = (uint32_t)id < (uint32_t)a.n;
            float dot = 0.f;
            if (ok) {
                for (int b = t; b * MX_BLOCK < a.d; b += 4) {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.codes + ((size_t)id * a.groups * 64 + b * 16)));
                    const float s = mx_scale(__ldg(a.scales + mx_scale_at(id, a.groups, b >> 2) + t));
                    float sum = 0.f;
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t h[4];
                        mx_halves(ws[k], h);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 f = half_pair(h[i]);
                            const int col = b * MX_BLOCK + k * 8 + 2 * i;
                            if (col < a.d) sum = fmaf(f.x, (float)x[col], sum);
                            if (col + 1 < a.d) sum = fmaf(f.y, (float)x[col + 1], sum);
                        }
                    }
                    dot = fmaf(sum, s, dot);
                }
            }
            dot += __shfl_xor_sync(0xFFFFFFFFu, dot, 1);
            dot += __shfl_xor_sync(0xFFFFFFFFu, dot, 2);
            if (t == 0 && c < last) {
                float v = dot;
                if (!ok) v = __int_as_float(0x7FFFFFFF);
                else if (a.metric == MX_COSINE) v = dot * inverse_length(__ldg(a.norms + id)) * inverse_length(q2);
                else if (a.metric == MX_EUCLIDEAN) v = fmaf(2.f, dot, -q2) - __ldg(a.norms + id);
                a.out[c] = finite_or_nan(v);
            }
        }
        at = last;
    }
}

// ------------------------------------------------------------------------------------------
// Many candidates: on the tensor cores.  An MMA of 4-bit operands needs the query in 4 bits too, so a query becomes a sum of slices, each a row in
// microscaled 4 bits: slice j of a block holds the rest behind slice j - 1, to the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6} times 2^(E - 2 j).  The rest is exact, and each slice takes two
// bits at least, so that a query of float32 values within a factor of 2^10 of one another in a block is the sum of about 18 slices, one of bytes that of five: nothing is rounded
// off.  Sixteen, 32, 48 or 64 slices of a query are the N side of the MMAs; those beyond 64 would be below 2^-126 of the block's largest value.  A scale is no less than 2^-127: a query whose
// values are all below 2^-64 is multiplied by a power of two that brings the largest there, and its scores are by that less, so that no bit above 2^-63 of a query's largest value is
// lost (and no sum of such a query can pass float32, whatever the rows' scales).  The M side are 128 candidates of a list, whose codes
// and scales are gathered by cp.async to where the MMAs take them, and the score is the sum of the accumulator's columns.  No code is unpacked by an instruction:
// 180M candidates of 128 values 12.0 -> 3.7 ms.  Of 100,000 rows, which lie in L2, they take 2.5 ms: what a warp does for a
// tile; of a million the gather takes longer: 172 bytes a candidate from L2 in pieces of 32 and 64 bytes, 7.7 TB/s (3.1 ms without its norm), with L2's tags at 36 %, its sectors at
// 22 and issue at 51: warps wait for gathers and for one another.  Codes gathered by TMA took 3.4 ms in either case.
//
// One persistent CTA per SM.  Warps 0 - 11 gather (four a stage), 12 loads slices, 13 - 18 issue MMAs (a tile each: what a warp does for one takes 1,300 cycles), 19 - 30 epilogue (four a tile).
// All walk the same tiles: a CTA has those that begin in its share of the positions, where each list counts for 128 more than it has.
// ------------------------------------------------------------------------------------------
constexpr int MXS_SLICES = 64, MXS_B_BYTES = MXS_SLICES * 64 + MX_TILE_BYTES;  // of a query and a group: codes, swizzled, and scales
constexpr int MXS_ROWS = 128, MXS_A_BYTES = MXS_ROWS * 64 + MX_TILE_BYTES;
constexpr int MXS_STAGES = 18, MXS_B_SLOTS = 12, MXS_KEPT = 4;                 // groups up to which all slices of a list stay while it lasts
constexpr int MXS_SETS = 3, MXS_GATHER_WARPS = 4 * MXS_SETS, MXS_MMA_WARPS = 6, MXS_EPI_WARPS = 4 * MXS_SETS, MXS_THREADS = 32 * (MXS_GATHER_WARPS + MXS_MMA_WARPS + 1 + MXS_EPI_WARPS);
constexpr int MXS_ACCS = 6, MXS_SF_COL = MXS_ACCS * MXS_SLICES, MXS_SF_SLOTS = (512 - MXS_SF_COL) / 8 / MXS_MMA_WARPS;  // slots of each
constexpr int MXS_SMEM = MXS_STAGES * MXS_A_BYTES + MXS_B_SLOTS * MXS_B_BYTES + 1024 + 1024;

// What is known of a query's slices, in a word: their number (a multiple of 16), and the power of two that they have been multiplied by.
__device__ __forceinline__ int mxs_count(int word) { return word & 255; }
__device__ __forceinline__ float mxs_down(int word) { return __uint_as_float((uint32_t)(127 - (word >> 8)) << 23); }

// Slices of queries first .. first + gridDim.x - 1, a CTA each: of[q] [groups][MXS_B_BYTES], that word and the squared length.
template <typename T>
__global__ void __launch_bounds__(128) mx_slices_kernel(const T* __restrict__ Q, int64_t ldq, int d, int groups, int first, uint8_t* __restrict__ slices,
                                                        int* __restrict__ counts, float* __restrict__ norms, KernelBefore before) {
    behind_kernel_before(Q, slices, counts, norms, before);
    __shared__ int s_need[4];
    __shared__ uint32_t s_top[4];
    __shared__ float s_norm[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* __restrict__ q = Q + (int64_t)(first + blockIdx.x) * ldq;
    auto value = [&](int block) {
        const int c = block * MX_BLOCK + lane;
        return c < d ? (float)__ldcg(q + c) : 0.f;
    };
    uint32_t top = 0;
    for (int b = warp; b < groups * 4; b += 4) top = max(top, __float_as_uint(value(b)) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
    top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    const int exponent_of_top = top >= 0x800000u ? (int)(top >> 23) - 127 : -118 - __clz((int)top);  // of the smallest ones, too
    const int shift = top != 0 && exponent_of_top < -64 ? -64 - exponent_of_top : 0;
    const float up = __uint_as_float((uint32_t)(127 + shift) << 23);
    // exponent of a block's first slice (of a value that is not finite: no slices, and a scale that is NaN)
    auto exponent = [&](float v, bool& bad) {
        const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v) & 0x7FFFFFFFu);
        bad = m >= 0x7F800000u;
        return max((int)(m >> 23) - 129, -127);
    };
    int need = 1;
    float norm = 0.f;
    for (int b = warp; b < groups * 4; b += 4) {
        float v = value(b);
        norm = fmaf(v, v, norm);
        v *= up;
        bool bad;
        const int e = exponent(v, bad);
        // the lowest bit of the block's values, as an exponent
        const uint32_t bits = __float_as_uint(v) & 0x7FFFFFFFu, fraction = (bits & 0x7FFFFFu) | (bits >= 0x800000u ? 0x800000u : 0u);
        int low = bits ? max((int)(bits >> 23), 1) - 150 + __ffs((int)fraction) - 1 : 1 << 20;
        low = __reduce_min_sync(0xFFFFFFFFu, low);
        if (!bad && low < 1 << 20) need = max(need, (e - low) / 2 + 2);  // the last one's values are multiples of two in units of its scale, and below eight
    }
    for (int o = 16; o; o >>= 1) norm += __shfl_xor_sync(0xFFFFFFFFu, norm, o);
    if (lane == 0) {
        s_need[warp] = need;
        s_norm[warp] = norm;
    }
    __syncthreads();
    need = max(max(s_need[0], s_need[1]), max(s_need[2], s_need[3]));
    const int count = min((need + 15) & ~15, MXS_SLICES);
    if (threadIdx.x == 0) {
        counts[blockIdx.x] = count | shift << 8;
        const float all = (s_norm[0] + s_norm[1]) + (s_norm[2] + s_norm[3]);
        norms[blockIdx.x] = all == 0.f && top != 0 ? MX_LEAST : all;
    }
    for (int b = warp; b < groups * 4; b += 4) {
        uint8_t* const to = slices + ((size_t)blockIdx.x * groups + (b >> 2)) * MXS_B_BYTES;
        float rest = value(b) * up;
        bool bad;
        int e = exponent(rest, bad);
        for (int j = 0; j < count; ++j, e -= 2) {
            uint32_t code = 0;
            if (!bad && e >= -127) {  // below that a block has no scale: what is left is less than 2^-125
                float y[8] = {rest * __uint_as_float((uint32_t)(127 - e) << 23), 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                code = mx_codes(y) & 15u;
                uint32_t h[4];
                mx_halves(code, h);
                rest = fmaf(-half_pair(h[0]).x, mx_scale((uint32_t)(e + 127)), rest);
            }
            uint32_t word = code << (4 * (lane & 7));
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
            if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(to + j * 64 + (((b & 3) ^ ((j >> 1) & 3)) << 4) + (lane >> 3) * 4) = word;
            if (lane == 0) to[MXS_SLICES * 64 + (j & 31) * 16 + (j >> 5) * 4 + (b & 3)] = (uint8_t)(bad ? 255 : max(e, -127) + 127);
        }
    }
}

struct MxScoreBatch {
    MxScoreArgs a;
    const uint8_t* slices;
    const int* counts;
    const float* q_norms;
    int* d_error;
    int first, last;  // queries
    bool kept;        // MXS_KEPT
    int warps;        // that issue MMAs
    int stages;       // of the ring, a multiple of the sets and, where there are more warps than one, of their tiles' stages
    int lists;        // kept ones, or slots for stages
};

// The tiles of a CTA, list by list.  Most steps stay in a list and cost an add and a subtraction: whole warps wait for what a warp does between its waits.
struct MxTiles {
    const int64_t* offsets;
    int64_t at, end, stop, total;  // at: first position of the tile; end: of the list; positions count as at + 128 q, and the CTA has those below stop
    int q, last, left;             // left: tiles of the list from this one on
    uint32_t nth;                  // of the lists that have tiles here
    __device__ __forceinline__ int64_t offset(int i) const { return min(max(__ldg(offsets + i), (int64_t)0), total); }
    __device__ __forceinline__ MxTiles(const MxScoreBatch& b) : offsets(b.a.offsets), total(b.a.total), last(b.last), nth(0) {
        const int64_t from = offset(b.first) + (int64_t)MXS_ROWS * b.first, to = max(offset(last) + (int64_t)MXS_ROWS * last, from);
        const int64_t share = (to - from) / gridDim.x + 1;
        const int64_t start = from + share * blockIdx.x;
        stop = min(start + share, to);
        int lo = b.first, hi = last;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (offset(mid) + (int64_t)MXS_ROWS * mid <= start) lo = mid;
            else hi = mid;
        }
        q = lo;
        const int64_t begin = offset(q);
        at = begin + (max(start - begin - (int64_t)MXS_ROWS * q, (int64_t)0) + MXS_ROWS - 1) / MXS_ROWS * MXS_ROWS;
        end = offset(q + 1);
        settle();
    }
    // Counts the list's tiles; goes on to one that has some.
    __device__ __forceinline__ void settle() {
        while (true) {
            const int64_t to = min(end, stop - (int64_t)MXS_ROWS * q);
            left = to > at ? (int)((to - at + MXS_ROWS - 1) / MXS_ROWS) : 0;
            if (left) return;
            if (++q >= last) return;
            at = offset(q);
            if (at + (int64_t)MXS_ROWS * q >= stop) {
                q = last;
                return;
            }
            end = offset(q + 1);
        }
    }
    __device__ __forceinline__ bool live() const { return left > 0; }
    __device__ __forceinline__ void next(int n) {
        while (n >= left) {
            if (!left) return;
            n -= left;
            ++nth;
            at = end;
            settle();
        }
        at += (int64_t)n * MXS_ROWS;
        left -= n;
    }
    __device__ __forceinline__ void next_list() { next(left); }
};

// A place in a ring of `n`, and the parity of the phase that is waited for there.  Counted on, not divided: a division costs a warp more than its wait.
struct MxRing {
    uint32_t at, parity;
    __device__ __forceinline__ void on(uint32_t by, uint32_t n) {  // by no more than n
        at += by;
        if (at >= n) {
            at -= n;
            parity ^= 1u;
        }
    }
};

__device__ __forceinline__ void copy_async16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// Launched as usual: it reads ids, offsets and scales (4 bytes by cp.async) by L1.
__global__ void __launch_bounds__(MXS_THREADS, 1) mx_score_tc_kernel(MxScoreBatch b) {
    extern __shared__ unsigned char mxs_smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mxs_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* s_b = base + MXS_STAGES * MXS_A_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_b + MXS_B_SLOTS * MXS_B_BYTES);
    uint64_t* empty = full + MXS_STAGES;
    uint64_t* b_full = empty + MXS_STAGES;
    uint64_t* b_empty = b_full + MXS_B_SLOTS;
    uint64_t* acc_full = b_empty + MXS_B_SLOTS;
    uint64_t* acc_empty = acc_full + MXS_ACCS;
    uint64_t* drained = acc_empty + MXS_ACCS;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    uint32_t* s_fills = s_tmem + 2;  // slots of slices that have been loaded
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const MxScoreArgs& a = b.a;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MXS_STAGES; ++s) {
            mbar_init(&full[s], 4);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < MXS_B_SLOTS; ++s) {
            mbar_init(&b_full[s], 1);
            mbar_init(&b_empty[s], (uint32_t)b.warps);  // a list's slices have gone by, or a stage's
        }
        for (int s = 0; s < MXS_ACCS; ++s) {
            mbar_init(&acc_full[s], 1);
            mbar_init(&acc_empty[s], 4);
        }
        mbar_init(drained, MXS_MMA_WARPS);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MXS_GATHER_WARPS + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    MxTiles tiles(b);

    if (warp < MXS_GATHER_WARPS) {
        // A set takes every third stage, so that none of its waits for a stage is more than one phase of the barrier behind.
        const int set = warp >> 2, r0 = (warp & 3) * 32, step = a.groups == 1 ? MXS_SETS : 1;
        const uint32_t ring = (uint32_t)b.stages;
        auto id_of = [&](const MxTiles& t) { return t.live() && t.at + r0 + lane < t.end ? __ldg(a.ids + t.at + r0 + lane) : -1; };
        const uint32_t pitch = (uint32_t)a.groups * 64u;
        const uint32_t to0 = smem_u32(base) + (r0 + (lane >> 2)) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);  // eight rows by four pieces of 16 bytes
        const uint32_t scale0 = smem_u32(base) + MXS_ROWS * 64 + lane * 16 + (warp & 3) * 4;
        uint32_t in_flight = 0;
        MxRing stage{(uint32_t)set, 1u}, landing{(uint32_t)set, 0u};
        auto land = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[landing.at]);
            landing.on(MXS_SETS, ring);
            --in_flight;
        };
        if (step > 1) tiles.next(set);
        int32_t id = id_of(tiles);
        bool live = true;
        uint32_t first = step > 1 ? 0u : (uint32_t)set;  // group of the tile that is the set's
        while (tiles.live() && live) {
            tiles.next(step);
            const int32_t id_next = id_of(tiles);  // on its way while the rows of this tile are asked for
            if ((uint32_t)id >= (uint32_t)a.n) id = -1;
            const uint8_t* scales = a.scales + (id >= 0 ? mx_scale_at(id, a.groups, 0) : 0);
            uint32_t g = first;
            for (; g < (uint32_t)a.groups; g += MXS_SETS) {
                if (!mbar_wait_warp(&empty[stage.at], stage.parity, s_abort, b.d_error)) { live = false; break; }
                const uint32_t to = stage.at * MXS_A_BYTES;
                const uint8_t* codes = a.codes + g * 64 + (lane & 3) * 16;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t from = __shfl_sync(0xFFFFFFFFu, id, i * 8 + (lane >> 2));
                    if (from >= 0) copy_async16(to0 + to + i * 512, codes + (uint64_t)(uint32_t)from * pitch);
                }
                if (id >= 0) copy_async4(scale0 + to, scales + g * MX_TILE_BYTES);
                asm volatile("cp.async.commit_group;" ::: "memory");
                stage.on(MXS_SETS, ring);
                ++in_flight;
                // of all sets fewer than the ring has, or the MMAs could wait for a stage that waits for them
                if (ring == MXS_STAGES && in_flight > 5) {
                    asm volatile("cp.async.wait_group 5;" ::: "memory");
                    land();
                } else if (ring != MXS_STAGES && in_flight > 3) {
                    asm volatile("cp.async.wait_group 3;" ::: "memory");
                    land();
                }
            }
            if (step == 1) first = g - (uint32_t)a.groups;
            id = id_next;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        while (in_flight) land();
    } else if (warp == MXS_GATHER_WARPS) {
        if (lane == 0) {
            uint32_t slot = 0, parity = 1, fills = 0;
            bool live = true;
            while (tiles.live() && live) {
                const int q = tiles.q - b.first;
                const uint32_t codes = (uint32_t)mxs_count(__ldcg(b.counts + q)) * 64u;
                for (int g = 0; g < a.groups; ++g) {
                    if (!b.kept || g == 0) {
                        if (!mbar_wait(&b_empty[slot], parity, s_abort, b.d_error)) { live = false; break; }
                        mbar_expect_tx(&b_full[slot], (codes + MX_TILE_BYTES) * (b.kept ? (uint32_t)a.groups : 1u));
                        ++fills;
                    }
                    unsigned char* to = s_b + (b.kept ? slot * a.groups + g : slot) * MXS_B_BYTES;
                    const uint8_t* from = b.slices + ((size_t)q * a.groups + g) * MXS_B_BYTES;
                    bulk_load(to, from, codes, &b_full[slot]);
                    bulk_load(to + MXS_SLICES * 64, from + MXS_SLICES * 64, MX_TILE_BYTES, &b_full[slot]);
                    if ((!b.kept || g == a.groups - 1) && ++slot == (uint32_t)b.lists) { slot = 0; parity ^= 1u; }
                }
                if (b.kept) tiles.next_list();
                else tiles.next(1);
            }
            *s_fills = fills;
        }
    } else if (warp <= MXS_GATHER_WARPS + MXS_MMA_WARPS) {
        // Tiles go to the warps in turn where the ring holds a multiple of the warps' tiles: each barrier of a stage or an accumulator is waited for by the same warp then.  Longer
        // rows are one warp's.
        const uint32_t w = warp - MXS_GATHER_WARPS - 1, warps = (uint32_t)b.warps, ring = (uint32_t)b.stages, lists = (uint32_t)b.lists;
        uint32_t sf = 0;
        bool live = w < warps;
        uint32_t seen = 0;  // lists that this warp has nothing more to do with
        MxRing list{0u, 0u}, stage{w * a.groups, 0u}, acc{w, 1u};
        auto leave = [&]() {
            if (b.kept)
                for (; seen < tiles.nth && live; ++seen) {  // also those of which it had no tile, so that none of its waits is more than a phase behind
                    live = mbar_wait_warp(&b_full[list.at], list.parity, s_abort, b.d_error);
                    if (live) tc_commit_warp(&b_empty[list.at]);
                    list.on(1, lists);
                }
        };
        tiles.next((int)w);
        leave();
        int q = -1, count = 0;
        while (tiles.live() && live) {
            if (tiles.q != q) {
                q = tiles.q;
                count = mxs_count(__ldcg(b.counts + q - b.first));
            }
            const uint32_t id0 = mx_idesc(count, 0), id1 = mx_idesc(count, 2);
            if (!mbar_wait_warp(&acc_empty[acc.at], acc.parity, s_abort, b.d_error)) break;
            const uint32_t d_tmem = tmem + acc.at * MXS_SLICES;
            for (int g = 0; g < a.groups; ++g) {
                if ((!b.kept || g == 0) && !mbar_wait_warp(&b_full[list.at], list.parity, s_abort, b.d_error)) { live = false; break; }
                if (!mbar_wait_warp(&full[stage.at], stage.parity, s_abort, b.d_error)) { live = false; break; }
                // what the gathering threads copied, for the MMAs; a fence of theirs would wait for the copies that they have in flight
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_after();
                const uint32_t st = smem_u32(base) + stage.at * MXS_A_BYTES;
                const uint32_t sb = smem_u32(s_b) + (b.kept ? list.at * a.groups + g : list.at) * MXS_B_BYTES;
                const uint64_t da = mx_tile_desc<64>(st), db = mx_tile_desc<64>(sb);
                const uint32_t sfa = tmem + MXS_SF_COL + (w * MXS_SF_SLOTS + sf) * 8, sfb = sfa + 4;
                sf = (sf + 1) % MXS_SF_SLOTS;
                tc_copy_scales(sfa, mx_scale_desc(st + MXS_ROWS * 64));
                tc_copy_scales(sfb, mx_scale_desc(sb + MXS_SLICES * 64));
                tc_mma_mxf4(d_tmem, da, db, id0, sfa, sfb, g != 0);
                tc_mma_mxf4(d_tmem, da + 2, db + 2, id1, sfa, sfb, 1u);
                tc_commit_warp(&empty[stage.at]);
                stage.on(1, ring);
                if (!b.kept) {
                    tc_commit_warp(&b_empty[list.at]);
                    list.on(1, lists);
                }
            }
            if (!live) break;
            tc_commit_warp(&acc_full[acc.at]);
            acc.on(warps, MXS_ACCS);
            stage.on((warps - 1) * a.groups, ring);
            tiles.next((int)warps);
            leave();
        }
    } else {
        // An id takes as long to come as several tiles take, and the norm that it names as long again: ids are asked for two of this set's tiles ahead, norms one.
        struct Ahead {
            int64_t at;  // of this lane's candidate, or -1
            int32_t id;
            int q;       // or -1
            float norm;
        };
        const int set = (warp - MXS_GATHER_WARPS - MXS_MMA_WARPS - 1) >> 2, quarter = warp & 3;
        tiles.next(set);
        auto take = [&]() {
            Ahead t;
            t.at = tiles.live() && tiles.at + quarter * 32 + lane < tiles.end ? tiles.at + quarter * 32 + lane : -1;
            t.id = t.at >= 0 ? __ldg(a.ids + t.at) : -1;
            t.q = tiles.live() ? tiles.q - b.first : -1;
            t.norm = 0.f;
            tiles.next(MXS_SETS);
            return t;
        };
        auto norm_of = [&](Ahead& t) {
            if (a.metric != MX_DOT && (uint32_t)t.id < (uint32_t)a.n) t.norm = __ldcg(a.norms + t.id);
        };
        Ahead now = take(), next = take();
        norm_of(now);
        bool live = true;
        int q = -1, count = 0;
        float q_term = 0.f, down = 1.f;
        for (MxRing acc{(uint32_t)set, 0u}; now.q >= 0; acc.on(MXS_SETS, MXS_ACCS)) {
            const Ahead later = take();
            norm_of(next);
            if (now.q != q) {
                q = now.q;
                const int word = __ldcg(b.counts + q);
                count = mxs_count(word);
                down = mxs_down(word);
                q_term = norm_term(a.metric, __ldcg(b.q_norms + q));
            }
            if (live) live = mbar_wait_warp(&acc_full[acc.at], acc.parity, s_abort, b.d_error);
            tc_fence_after();
            float v = 0.f;
            if (live) {
                const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + acc.at * MXS_SLICES;
                for (int c = count - 16; c >= 0; c -= 16) {  // the small slices first
                    uint32_t r[16];
                    tc_ld16(from + c, r);
                    tc_ld_wait();
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = __uint_as_float(r[2 * j + 1]) + __uint_as_float(r[2 * j]);
                    v += (w[7] + w[6]) + (w[5] + w[4]);
                    v += (w[3] + w[2]) + (w[1] + w[0]);
                }
                v *= down;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc.at]);
            if (a.metric == MX_COSINE) v = v * inverse_length(now.norm) * q_term;
            else if (a.metric == MX_EUCLIDEAN) v = fmaf(2.f, v, -q_term) - now.norm;
            if (now.at >= 0) a.out[now.at] = (uint32_t)now.id < (uint32_t)a.n && live ? finite_or_nan(v) : __int_as_float(0x7FFFFFFF);
            now = next;
            next = later;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*s_abort) {  // all roles are done: what they issued may not be (the gathering warps have waited for their copies)
        if (threadIdx.x == 32 * MXS_GATHER_WARPS) mbar_wait_landed(b_full, (uint32_t)b.lists, *s_fills);
        if (warp > MXS_GATHER_WARPS && warp <= MXS_GATHER_WARPS + MXS_MMA_WARPS) {
            tc_commit_warp(drained);
            mbar_wait_landed(drained, 1, 1);
        }
        __syncthreads();
    }
    if (warp == MXS_GATHER_WARPS + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Whether the kernel above, in one launch, is done sooner: it takes 0.08 us for a thousand groups of candidates, the tensor cores' 0.02 us, and 12 ns for a list (100 lists of 4,000 of 128
// values 36 us and 39, of 16,000 124 and 67; 10,000 lists of 160 137 and 157).
inline bool mx_score_few(int64_t total, int groups, int nq) { return total * groups < 200ll * (1000 + nq); }
// Queries whose slices lie in the workspace at a time.
inline int mx_score_batch(int nq, int groups) {
    const size_t per = (size_t)groups * MXS_B_BYTES;
    return (int)std::min<size_t>((size_t)nq, std::max<size_t>(1, ((size_t)64 << 20) / per));
}
inline size_t mx_score_workspace(int nq, int d, int64_t total) {
    if (mx_score_few(total, mx_groups(d), nq)) return 0;
    const size_t batch = (size_t)mx_score_batch(nq, mx_groups(d));
    return batch * mx_groups(d) * MXS_B_BYTES + batch * 8;
}

template <typename T>
inline void mx_score(const CtxPtr& c, const T* Q, const MxScoreArgs& a, void* workspace, int* d_error, cudaStream_t stream) {
    if (mx_score_few(a.total, a.groups, a.nq)) {
        const int per = 8 * (int)std::min<int64_t>(8, std::max<int64_t>(1, a.total / (8 * 32 * c->sm_count)));  // 32 warps for an SM first
        mx_score_kernel<T><<<(unsigned)ceil_div((size_t)a.total, 8 * (size_t)per), 256, 0, stream>>>(Q, a, per);
        KERNEL_CHECK();
        return;
    }
    const int batch = mx_score_batch(a.nq, a.groups);
    uint8_t* const slices = static_cast<uint8_t*>(workspace);
    int* const counts = reinterpret_cast<int*>(slices + (size_t)batch * a.groups * MXS_B_BYTES);
    float* const norms = reinterpret_cast<float*>(counts + batch);
    static thread_local uint64_t ready = 0;  // devices whose limit is set
    if (c->device >= 64 || !(ready >> c->device & 1)) {
        CU_CHECK(cudaFuncSetAttribute(mx_score_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MXS_SMEM));
        if (c->device < 64) ready |= 1ull << c->device;
    }
    for (int q = 0; q < a.nq; q += batch) {
        MxScoreBatch b{a, slices, counts, norms, d_error, q, std::min(q + batch, a.nq)};
        b.kept = a.groups <= MXS_KEPT;
        b.warps = !b.kept ? 1 : a.groups == 1 ? MXS_MMA_WARPS : MXS_MMA_WARPS / 2;
        b.stages = MXS_STAGES / (b.warps * a.groups) ? MXS_STAGES / (b.warps * a.groups) * (b.warps * a.groups) : MXS_STAGES;
        if (!b.kept) b.stages = MXS_STAGES;
        b.lists = b.kept ? MXS_B_SLOTS / a.groups : MXS_B_SLOTS;
        launch_next(stream, mx_slices_kernel<T>, (size_t)(b.last - q), 128u, 0, Q, a.ldq, a.d, a.groups, q, slices, counts, norms);
        KERNEL_CHECK();
        mx_score_tc_kernel<<<(unsigned)c->sm_count, MXS_THREADS, MXS_SMEM, stream>>>(b);
        KERNEL_CHECK();
    }
}

}  // namespace culsh_b200
