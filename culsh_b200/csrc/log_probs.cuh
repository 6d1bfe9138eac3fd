// Log probabilities over scores: for every row of a matrix, or list of a CSR result, of scores s and z = s / temperature
//   lse = log sum exp z,   log p of a given entry = z - lse,   entropy = lse - sum p z,   and the k most likely entries,
// and the gradient of the first and the second with respect to s:  ds_i = (g ([i = given] - p_i) - h p_i (log p_i + entropy)) / temperature.
//
// One pass over the scores.  A warp takes chunks of 512 neighbouring entries, 16 to a lane, and keeps the largest score so far m and two sums relative to it,
//   l = sum 2^d,   e = sum d 2^d,   d = (s - m) log2(e) / temperature,
// in 32 bits; entropy = log l - log(2) e / l.  A larger m rescales both.  Parts (m, l, e) are joined in a fixed order, so results do not depend on how CTAs are scheduled.
// d is cut at -10,000, far below where 2^d is 0, so that an entry of -inf is 0 in both sums; m starts at the lowest finite value for the same reason.  NaN and +inf reach the sums and make
// them NaN.
//
// The k largest come from the chunks' maxima, which the pass leaves behind: the k largest entries (the earlier of equal ones first) lie in the k chunks whose
// maxima are the largest (the earlier of equal ones first), as every chunk before another in that order has an entry that comes before all of the other's.  So k chunks are read again,
// whatever the scores are.
//
// Rows begin anywhere: positions count from a 16-byte boundary at or in front of the array, chunks begin at multiples of 512 of those, and the first and the last one of a row
// load entry by entry.
#pragma once

#include "mx_score.cuh"

namespace culsh_b200 {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_PER_LANE = 16, LP_CHUNK = 32 * LP_PER_LANE;
constexpr int LP_CHUNKS = 1024;                 // maxima that a CTA keeps of a row; a longer row's stand for several chunks each
constexpr int LP_STEP = 4 * LP_THREADS;         // entries that are looked at before the collected ones are counted
constexpr int LP_KEYS = 2 * LP_STEP, LP_MAX_K = 128;
constexpr float LP_FLOOR = -10000.f;

// Where rows are: a matrix with rows `ld` apart and `cols` long, or lists.  Positions of row r: [begin, end).
struct LpRows {
    const int64_t* offsets;
    int64_t ld, cols, shift, total;  // shift: entries between the boundary and the array; total: entries of all lists
    __device__ __forceinline__ int64_t begin(int r) const {
        return (offsets ? min(max(__ldg(offsets + r), (int64_t)0), total) : (int64_t)r * ld) + shift;
    }
    __device__ __forceinline__ int64_t end(int r) const {
        return offsets ? max(min(__ldg(offsets + r + 1), total) + shift, begin(r)) : (int64_t)r * ld + cols + shift;
    }
};

struct LpArgs {
    LpRows rows;
    const int32_t* ids;       // names of the entries of lists, ascending in each, or null
    const int64_t* targets;   // or null
    float* log_probs;         // or null, with targets
    float* entropy;
    float* lse;
    float* top_log_probs;     // or null, with k = 0
    int32_t* top_ids;
    int m, k;
    float c, inv_t;           // log2(e) / temperature, 1 / temperature
    // rows taken by several CTAs
    int64_t unit;             // positions of a CTA, a multiple of 512
    int units_per_row;        // of a matrix
    float4* parts;
    uint32_t* maxima;         // of the chunks; row r's from chunk_slot(r) on
};

// Order of scores as unsigned integers; NaN below everything, -0 as 0.
__device__ __forceinline__ uint32_t lp_order(float s) {
    const uint32_t b = __float_as_uint(s + 0.f);
    return s != s ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_score(uint32_t order) {
    return __uint_as_float((order & 0x80000000u) ? order & 0x7FFFFFFFu : ~order);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

struct LpPart {
    float m, l, e;
    static __device__ __forceinline__ LpPart none() { return {-3.402823466e38f, 0.f, 0.f}; }
    __device__ __forceinline__ void raise(float to, float c) {
        const float d = max_nan((m - to) * c, LP_FLOOR), f = exp2_fast(d);
        e = (e + l * d) * f;
        l *= f;
        m = to;
    }
    __device__ __forceinline__ void join(LpPart o, float c) {
        const float to = fmaxf(m, o.m);
        raise(to, c);
        o.raise(to, c);
        l += o.l;
        e += o.e;
    }
    __device__ __forceinline__ LpPart shuffled(int x) const {
        LpPart o;
        o.m = __shfl_xor_sync(0xFFFFFFFFu, m, x);
        o.l = __shfl_xor_sync(0xFFFFFFFFu, l, x);
        o.e = __shfl_xor_sync(0xFFFFFFFFu, e, x);
        return o;
    }
};

__device__ __forceinline__ float score_of(float s) { return s; }
__device__ __forceinline__ float score_of(__half s) { return __half2float(s); }
__device__ __forceinline__ float score_of(__nv_bfloat16 s) { return __bfloat162float(s); }

// Position of entry i of a lane's 16 in its chunk.
template <typename T>
__device__ __forceinline__ int lp_place(int lane, int i) {
    constexpr int V = 16 / sizeof(T);
    return ((i / V) * 32 + lane) * V + i % V;
}
// The lane's 16 scores of a chunk, -inf outside [begin, end).  `x`: position 0.
template <typename T>
__device__ __forceinline__ void lp_load(const T* __restrict__ x, int64_t chunk, int64_t begin, int64_t end, int lane, float (&s)[LP_PER_LANE]) {
    constexpr int V = 16 / sizeof(T);
    const int64_t p0 = chunk * LP_CHUNK;
    if (p0 >= begin && p0 + LP_CHUNK <= end) {
        uint4 w[LP_PER_LANE / V];
#pragma unroll
        for (int j = 0; j < LP_PER_LANE / V; ++j) w[j] = __ldg(reinterpret_cast<const uint4*>(x + p0) + j * 32 + lane);
#pragma unroll
        for (int i = 0; i < LP_PER_LANE; ++i) s[i] = score_of(reinterpret_cast<const T*>(&w[i / V])[i % V]);
    } else {
#pragma unroll
        for (int i = 0; i < LP_PER_LANE; ++i) {
            const int64_t p = p0 + lp_place<T>(lane, i);
            s[i] = p >= begin && p < end ? score_of(x[p]) : -INFINITY;
        }
    }
}

// A warp's chunks first, first + step, ... below last, all in one row; `leave(chunk, largest)` takes the maxima.
template <typename T, typename Leave>
__device__ __forceinline__ LpPart lp_chunks(const T* __restrict__ x, int64_t first, int64_t last, int step, int64_t begin, int64_t end, float c, int lane,
                                            Leave leave) {
    LpPart part = LpPart::none();  // m is the same in all lanes
    for (int64_t chunk = first; chunk < last; chunk += step) {
        float s[LP_PER_LANE];
        lp_load(x, chunk, begin, end, lane, s);
        float top = s[0];
#pragma unroll
        for (int i = 1; i < LP_PER_LANE; ++i) top = fmaxf(top, s[i]);
        if (top != top) top = -INFINITY;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        leave(chunk, top);
        if (top > part.m) part.raise(top, c);
        float l0 = 0.f, l1 = 0.f, e0 = 0.f, e1 = 0.f;
#pragma unroll
        for (int i = 0; i < LP_PER_LANE; i += 2) {
            const float d0 = max_nan((s[i] - part.m) * c, LP_FLOOR), d1 = max_nan((s[i + 1] - part.m) * c, LP_FLOOR);
            const float p0 = exp2_fast(d0), p1 = exp2_fast(d1);
            l0 += p0;
            l1 += p1;
            e0 = fmaf(p0, d0, e0);
            e1 = fmaf(p1, d1, e1);
        }
        part.l += l0 + l1;
        part.e += e0 + e1;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        part.l += __shfl_xor_sync(0xFFFFFFFFu, part.l, o);
        part.e += __shfl_xor_sync(0xFFFFFFFFu, part.e, o);
    }
    return part;
}

struct LpShared {
    uint64_t keys[LP_KEYS];
    uint32_t maxima[LP_CHUNKS];
    LpPart parts[LP_WARPS];
    int count;
    int64_t target;  // position of the given entry, or -1
};

// The CTA's part from its warps', in the order of the warps; for all threads.
__device__ __forceinline__ LpPart lp_join_warps(LpShared& sh, const LpPart& mine, float c) {
    if ((threadIdx.x & 31) == 0) sh.parts[threadIdx.x >> 5] = mine;
    __syncthreads();
    LpPart all = sh.parts[0];
#pragma unroll
    for (int w = 1; w < LP_WARPS; ++w) all.join(sh.parts[w], c);
    return all;
}

// Sorts keys[0, n), n a power of two, the largest first.
__device__ __forceinline__ void lp_sort(uint64_t* keys, int n) {
    for (int size = 2; size <= n; size *= 2) {
        for (int stride = size / 2; stride; stride >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += LP_THREADS) {
                const int at = 2 * i - (i & (stride - 1));
                const uint64_t a = keys[at], b = keys[at + stride];
                if ((a < b) == ((at & size) == 0)) {
                    keys[at] = b;
                    keys[at + stride] = a;
                }
            }
        }
    }
    __syncthreads();
}
// Sorts the collected keys, keeps the k largest.
__device__ __forceinline__ void lp_settle(LpShared& sh, int k) {
    __syncthreads();
    const int count = sh.count;
    int n = 2;
    while (n < count) n *= 2;
    for (int i = count + threadIdx.x; i < n; i += LP_THREADS) sh.keys[i] = 0;
    lp_sort(sh.keys, n);
    if (threadIdx.x == 0) sh.count = min(count, k);
    __syncthreads();
}
// The k largest keys of key(0 .. n - 1) that are at least `least`, sorted, into sh.keys; sh.count of them.  Keys differ from one another, 0 is none.
template <typename Key>
__device__ __forceinline__ void lp_largest(LpShared& sh, int64_t n, int k, uint64_t least, Key key) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int64_t i0 = 0; i0 < n; i0 += LP_STEP) {
        uint64_t v[LP_STEP / LP_THREADS];
#pragma unroll
        for (int j = 0; j < LP_STEP / LP_THREADS; ++j) {
            const int64_t i = i0 + j * LP_THREADS + threadIdx.x;
            v[j] = i < n ? key(i) : 0ull;
        }
#pragma unroll
        for (int j = 0; j < LP_STEP / LP_THREADS; ++j)
            if (v[j] && v[j] >= least) sh.keys[atomicAdd(&sh.count, 1)] = v[j];
        __syncthreads();
        if (sh.count > LP_KEYS - LP_STEP) {
            lp_settle(sh, k);
            if (sh.count == k) least = max(least, sh.keys[k - 1]);
        }
        __syncthreads();
    }
    lp_settle(sh, k);
}

// Position of the entry that `target` names in row r, or -1; by one warp.
__device__ __forceinline__ int64_t lp_find(const LpArgs& a, int64_t begin, int64_t end, int64_t target) {
    if (!a.ids) return target >= 0 && target < end - begin ? begin + target : -1;
    const int lane = threadIdx.x & 31;
    const int32_t* __restrict__ ids = a.ids - a.rows.shift;
    int64_t lo = begin, hi = end;  // ids below lo are smaller, at and behind hi larger
    while (hi > lo) {
        const int64_t step = (hi - lo + 31) / 32, p = lo + lane * step;
        const int32_t id = p < hi ? __ldg(ids + p) : 0x7FFFFFFF;
        const unsigned smaller = __ballot_sync(0xFFFFFFFFu, p < hi && id < target), same = __ballot_sync(0xFFFFFFFFu, p < hi && id == target);
        if (same) return lo + (int64_t)(__ffs((int)same) - 1) * step;
        const int n = __popc(smaller);  // the first n probes
        if (!n) return -1;
        hi = min(hi, lo + n * step);
        lo = lo + (n - 1) * step + 1;
    }
    return -1;
}

// What a row's result is made of, by the whole CTA.  `maxima`: orders of the largest scores of groups of 512 << wide entries from first_chunk on.
template <typename T>
__device__ __forceinline__ void lp_finish(const T* __restrict__ x, const LpArgs& a, LpShared& sh, int row, int64_t begin, int64_t end, LpPart all,
                                          const uint32_t* maxima, int64_t first_chunk, int groups, int wide) {
    const float log_l = logf(all.l);
    const float z_max = all.m * a.inv_t;
    float lse = z_max + log_l, entropy = log_l - 0.69314718056f * (all.e / all.l);
    if (all.l == 0.f || lse == -INFINITY) {  // nothing, or nothing that is not masked
        lse = -INFINITY;
        entropy = 0.f;
    }
    // relative to the largest, as the sums are: nothing is lost where z is large
    auto log_p = [&](float s) { return s * a.inv_t == -INFINITY ? -INFINITY : lse == -INFINITY ? NAN : (s - all.m) * a.inv_t - log_l; };
    if (threadIdx.x == 0) {
        a.lse[row] = lse;
        a.entropy[row] = entropy;
        if (a.targets) a.log_probs[row] = sh.target < 0 ? -INFINITY : log_p(score_of(x[sh.target]));
    }
    if (!a.k) return;
    lp_largest(sh, groups, a.k, 0, [&](int64_t g) { return (uint64_t)maxima[g] << 32 | (0xFFFFFFFFu - (uint32_t)g); });
    const int kept = sh.count;
    __shared__ uint32_t s_groups[LP_MAX_K];
    for (int i = threadIdx.x; i < kept; i += LP_THREADS) s_groups[i] = 0xFFFFFFFFu - (uint32_t)sh.keys[i];
    const uint64_t least = kept == a.k ? sh.keys[kept - 1] & 0xFFFFFFFF00000000ull : 0ull;  // k entries are as large as the k-th of the maxima
    const int shift = 9 + wide;
    lp_largest(sh, (int64_t)kept << shift, a.k, least, [&](int64_t i) {
        const int64_t p = ((first_chunk + ((int64_t)s_groups[i >> shift] << wide)) << 9) + (i & ((1ll << shift) - 1));
        if (p < begin || p >= end) return 0ull;
        const uint32_t o = lp_order(score_of(x[p]));
        return o ? (unsigned long long)o << 32 | (0xFFFFFFFFu - (uint32_t)(p - begin)) : 0ull;
    });
    for (int i = threadIdx.x; i < a.k; i += LP_THREADS) {
        float lp = -INFINITY;
        int32_t id = -1;
        if (i < sh.count) {
            const uint32_t at = 0xFFFFFFFFu - (uint32_t)sh.keys[i];
            const float s = lp_score((uint32_t)(sh.keys[i] >> 32));
            if (s * a.inv_t > -INFINITY) {
                lp = log_p(s);
                id = a.ids ? __ldg(a.ids - a.rows.shift + begin + at) : (int32_t)at;
            }
        }
        a.top_log_probs[(int64_t)row * a.k + i] = lp;
        a.top_ids[(int64_t)row * a.k + i] = id;
    }
}

// A CTA for each row.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_row_kernel(const T* __restrict__ x, LpArgs a) {
    __shared__ LpShared sh;
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t begin = a.rows.begin(row), end = a.rows.end(row);
    const int64_t first = begin / LP_CHUNK, last = end > begin ? (end + LP_CHUNK - 1) / LP_CHUNK : first;
    int wide = 0;
    while ((last - first + (1ll << wide) - 1) >> wide > LP_CHUNKS) ++wide;
    const int groups = (int)((last - first + (1ll << wide) - 1) >> wide);
    if (a.k) {
        for (int i = threadIdx.x; i < groups; i += LP_THREADS) sh.maxima[i] = 0;
        __syncthreads();
    }
    if (warp == 0 && a.targets) {
        const int64_t at = lp_find(a, begin, end, __ldg(a.targets + row));
        if (lane == 0) sh.target = at;
    }
    const LpPart mine = lp_chunks(x, first + warp, last, LP_WARPS, begin, end, a.c, lane, [&](int64_t chunk, float top) {
        if (a.k && lane == 0) atomicMax(&sh.maxima[(chunk - first) >> wide], lp_order(top));
    });
    const LpPart all = lp_join_warps(sh, mine, a.c);
    lp_finish(x, a, sh, row, begin, end, all, sh.maxima, first, groups, wide);
}

// Rows taken by several CTAs.  Slots of a row's units and chunks: blocks of `size` positions from the one that it begins in on; lists share the numbering of all
// positions, moved on by one for each list, so that no two share a slot.
__device__ __forceinline__ int64_t lp_slot(const LpArgs& a, int row, int64_t begin, int64_t size, int64_t per_row) {
    return a.rows.offsets ? begin / size + row : (int64_t)row * per_row;
}
__device__ __forceinline__ int64_t lp_chunks_per_row(const LpArgs& a) { return a.rows.cols / LP_CHUNK + 2; }

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_unit_kernel(const T* __restrict__ x, LpArgs a) {
    __shared__ LpShared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int row;
    int64_t nth;
    if (a.rows.offsets) {  // the last list whose first slot is not behind this one
        int lo = 0, hi = a.m;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (lp_slot(a, mid, a.rows.begin(mid), a.unit, 0) <= (int64_t)blockIdx.x) lo = mid;
            else hi = mid;
        }
        row = lo;
        nth = (int64_t)blockIdx.x - lp_slot(a, row, a.rows.begin(row), a.unit, 0);
    } else {
        row = (int)(blockIdx.x / (unsigned)a.units_per_row);
        nth = blockIdx.x - (unsigned)row * (unsigned)a.units_per_row;
    }
    const int64_t begin = a.rows.begin(row), end = a.rows.end(row);
    const int64_t from = max((begin / a.unit + nth) * a.unit, begin), to = min((begin / a.unit + nth + 1) * a.unit, end);
    if (from >= to) return;
    const int64_t slot = lp_slot(a, row, begin, LP_CHUNK, lp_chunks_per_row(a)), first = begin / LP_CHUNK;
    const LpPart mine = lp_chunks(x, from / LP_CHUNK + warp, (to + LP_CHUNK - 1) / LP_CHUNK, LP_WARPS, begin, end, a.c, lane, [&](int64_t chunk, float top) {
        if (a.k && lane == 0) a.maxima[slot + chunk - first] = lp_order(top);
    });
    const LpPart all = lp_join_warps(sh, mine, a.c);
    if (threadIdx.x == 0) a.parts[blockIdx.x] = make_float4(all.m, all.l, all.e, 0.f);
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_join_kernel(const T* __restrict__ x, LpArgs a) {
    __shared__ LpShared sh;
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t begin = a.rows.begin(row), end = a.rows.end(row);
    if (warp == 0 && a.targets) {
        const int64_t at = lp_find(a, begin, end, __ldg(a.targets + row));
        if (lane == 0) sh.target = at;
    }
    const int64_t units = end > begin ? (end - 1) / a.unit - begin / a.unit + 1 : 0, slot = lp_slot(a, row, begin, a.unit, a.units_per_row);
    LpPart mine = LpPart::none();
    for (int64_t u = threadIdx.x; u < units; u += LP_THREADS) {
        const float4 p = a.parts[slot + u];
        mine.join(LpPart{p.x, p.y, p.z}, a.c);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mine.join(mine.shuffled(o), a.c);
    const LpPart all = lp_join_warps(sh, mine, a.c);
    const int64_t first = begin / LP_CHUNK, last = end > begin ? (end + LP_CHUNK - 1) / LP_CHUNK : first;
    lp_finish(x, a, sh, row, begin, end, all, a.maxima + lp_slot(a, row, begin, LP_CHUNK, lp_chunks_per_row(a)), first, (int)(last - first), 0);
}

// ------------------------------------------------------------------------------------------
// Gradient
// ------------------------------------------------------------------------------------------
struct LpBackward {
    LpArgs f;
    const float* lse;
    const float* entropy;
    const float* g;         // of the log probabilities, or null
    const float* h;         // of the entropies, or null
    int64_t chunks;         // of all positions (lists), or of each row at most (a matrix)
};

// Constants of a row: ds = p (a - b log p) - g p, and g (1 - p) in place of -g p at the given entry; log p = z - lse, a = -h entropy / temperature, b = h / temperature,
// g by the temperature.
struct LpRowTerms {
    float lse, a, b, g;
    int64_t target;
};

template <typename T>
__device__ __forceinline__ LpRowTerms lp_row_terms(const T* __restrict__ x, const LpBackward& b, int row, int64_t begin, int64_t end) {
    LpRowTerms r;
    const float lse = __ldg(b.lse + row), h = b.h ? __ldg(b.h + row) : 0.f;
    float g = b.f.targets && b.g ? __ldg(b.g + row) : 0.f;
    r.target = -1;
    if (b.f.targets && b.g) {
        r.target = lp_find(b.f, begin, end, __ldg(b.f.targets + row));
        if (r.target < 0 || score_of(x[r.target]) * b.f.inv_t == -INFINITY) {  // a log probability of -inf stays where it is
            r.target = -1;
            g = 0.f;
        }
    }
    r.lse = lse;
    r.a = -h * __ldg(b.entropy + row) * b.f.inv_t;
    r.b = h * b.f.inv_t;
    r.g = g * b.f.inv_t;
    return r;
}
// 1 - p of an entry that is nearly certain is as exact as its log p: lists of one or two entries have hardly anything else.
__device__ __forceinline__ float lp_grad(const LpRowTerms& r, float s, float inv_t, bool given) {
    const float z = s * inv_t;
    if (z == -INFINITY) return 0.f;
    const float lp = max_nan(z - r.lse, LP_FLOOR), p = exp2_fast(lp * 1.4426950409f);  // no 0 times infinity for the lowest finite values
    return fmaf(p, fmaf(-r.b, lp, r.a), r.g * (given ? -expm1f(lp) : -p));
}
__device__ __forceinline__ void put_grad(float* o, float v) { *o = v; }
__device__ __forceinline__ void put_grad(__half* o, float v) { *o = __float2half_rn(v); }
__device__ __forceinline__ void put_grad(__nv_bfloat16* o, float v) { *o = __float2bfloat16_rn(v); }

// A warp for each chunk, and for each row in it.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_backward_kernel(const T* __restrict__ x, T* __restrict__ out, LpBackward b) {
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * LP_WARPS + (threadIdx.x >> 5);
    const LpRows& rows = b.f.rows;
    int row;
    int64_t chunk;
    if (rows.offsets) {
        if (n >= b.chunks) return;
        chunk = n;
        row = owner_of(rows.offsets, b.f.m, max(chunk * LP_CHUNK - rows.shift, (int64_t)0));
    } else {
        row = (int)(n / b.chunks);
        if (row >= b.f.m) return;
        chunk = rows.begin(row) / LP_CHUNK + n % b.chunks;
    }
    const int64_t p0 = chunk * LP_CHUNK, p1 = p0 + LP_CHUNK;
    for (; row < b.f.m; ++row) {
        const int64_t begin = rows.begin(row), end = rows.end(row);
        if (begin >= p1) break;
        const int64_t from = max(begin, p0), to = min(end, p1);
        if (from < to) {
            const LpRowTerms r = lp_row_terms(x, b, row, begin, end);
            T* const o = out + (rows.offsets ? -rows.shift : (int64_t)row * rows.cols - begin);
            for (int64_t p = from + lane; p < to; p += 32) {
                put_grad(o + p, lp_grad(r, score_of(x[p]), b.f.inv_t, p == r.target));
            }
        }
        if (!rows.offsets) break;
    }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
struct LpPlan {
    bool split = false;
    int64_t unit = 0, units = 0, chunks = 0;  // units and chunks of all rows
    int units_per_row = 0;
    size_t bytes() const { return split ? (size_t)units * sizeof(float4) + (size_t)chunks * sizeof(uint32_t) : 0; }
};

// Rows that fill the chip with a CTA each, and short ones, take one; others are taken by several.  total: entries of all lists.
inline LpPlan lp_plan(int m, int64_t cols, int64_t total, bool lists, int sm_count) {
    LpPlan p;
    const int64_t entries = lists ? total : (int64_t)m * cols, mean = m ? entries / m : 0;
    p.split = m < 4 * sm_count && mean > 16384;
    if (!p.split) return p;
    p.unit = 4096;
    while (p.unit < 32768 && entries / p.unit > 16ll * sm_count) p.unit *= 2;
    p.units_per_row = (int)(cols / p.unit + 2);
    p.units = lists ? (total + 16) / p.unit + m + 1 : (int64_t)m * p.units_per_row;
    p.chunks = lists ? (total + 16) / LP_CHUNK + m + 1 : (int64_t)m * (cols / LP_CHUNK + 2);
    return p;
}

template <typename T>
inline void log_probs(const CtxPtr& c, const T* scores, LpArgs a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    a.rows.shift = (int64_t)((uintptr_t)scores / sizeof(T) % V);
    const T* x = scores - a.rows.shift;
    const LpPlan p = lp_plan(a.m, a.rows.cols, a.rows.total, a.rows.offsets != nullptr, c->sm_count);
    if (!p.split) {
        log_probs_row_kernel<T><<<(unsigned)a.m, LP_THREADS, 0, stream>>>(x, a);
        KERNEL_CHECK();
        return;
    }
    if (workspace_bytes < p.bytes() || !workspace || ((uintptr_t)workspace & 15)) fail(CULSH_ERR_INVALID, "the workspace has to be %zu bytes, aligned to 16", p.bytes());
    if (p.units > 0x7FFFFFFFll) fail(CULSH_ERR_UNSUPPORTED, "%lld entries are too many for one call", (long long)a.rows.total);
    a.unit = p.unit;
    a.units_per_row = p.units_per_row;
    a.parts = static_cast<float4*>(workspace);
    a.maxima = reinterpret_cast<uint32_t*>(a.parts + p.units);
    log_probs_unit_kernel<T><<<(unsigned)p.units, LP_THREADS, 0, stream>>>(x, a);
    KERNEL_CHECK();
    log_probs_join_kernel<T><<<(unsigned)a.m, LP_THREADS, 0, stream>>>(x, a);
    KERNEL_CHECK();
}

template <typename T>
inline void log_probs_backward(const T* scores, T* out, LpBackward b, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    LpRows& r = b.f.rows;
    r.shift = (int64_t)((uintptr_t)scores / sizeof(T) % V);
    if (r.offsets) b.chunks = (int64_t)ceil_div((size_t)(r.total + r.shift), LP_CHUNK);
    else b.chunks = r.cols / LP_CHUNK + 2;
    const size_t grid = ceil_div(r.offsets ? (size_t)b.chunks : (size_t)b.chunks * b.f.m, LP_WARPS);
    if (grid > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "too many entries for one call");
    log_probs_backward_kernel<T><<<(unsigned)grid, LP_THREADS, 0, stream>>>(scores - r.shift, out, b);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
