// Log probabilities over scores: for every row of a matrix, or list of a CSR result, of scores s and z = s / temperature
//   lse = log sum exp z,   log p of a given entry = z - lse,   entropy = lse - sum p z,   and the k most likely entries,
// and the gradient of the first and the second with respect to s:  ds_i = (g ([i = given] - p_i) - h p_i (log p_i + entropy)) / temperature.
//
// One pass over the scores.  A warp takes chunks of 512 neighbouring entries, or 1,024 of 16 bits, and keeps the largest score so far m and two sums relative to it,
//   l = sum 2^d,   e = sum d 2^d,   d = (s - m) log2(e) / temperature,
// in 32 bits; entropy = log l - log(2) e / l.  A larger m rescales both.  d is one multiply-add, of s with the rounded product of m: what its rounding moved all d by is taken out of
// the sums at the end; of scores of 2^24 bits and more, where it would move d by whole bits, d is (s - m) log2(e) / temperature as it stands.  Parts (m, l, e) are joined in a fixed order, so results do not depend on how CTAs are scheduled.  An entry of -inf counts as a score so low that 2^d is 0 and d is finite;
// where m itself is that low, d is cut at -10,000 instead.  NaN and +inf reach the sums and make them NaN.
// Bound by HBM with 32 bits (1,000 x 1M 584 us, 6.8 TB/s).  With 16, five instructions and an exponential for an entry: HBM, issue and exponentials are at half each, with a quarter of the warps
// that an SM could hold (380 to 400 us, 5.2 TB/s; without the k largest 45 us less; a pass of eight instructions 579).  10,000 lists of 18,000 float32 205 us of 225 (the rest: targets that are in
// no list), 60 less without the k largest: what follows the pass is waits.
//
// The k largest: the pass leaves the largest entry of each thread and of each chunk behind.  The k-th largest of the threads' is a bound that at least k entries reach, and hardly more do (of 1M
// drawn at random and 256 threads about k + 1): only chunks that reach it are read again, and the entries that do are sorted, by score and then by place.  Where more entries are alike than
// there is room to sort at once, they are sorted in turns.
//
// Rows begin anywhere: positions count from a 16-byte boundary at or in front of the array, chunks begin at multiples of their length of those, and the first and the last one of a row
// load entry by entry.
#pragma once

#include "mx_score.cuh"

namespace culsh_b200 {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
// A lane has 64 bytes of a chunk, and 64 of the next one on their way.
template <typename T>
constexpr int LP_PER_LANE = 64 / sizeof(T);
template <typename T>
constexpr int LP_CHUNK = 32 * LP_PER_LANE<T>;
constexpr int LP_LEAST_CHUNK = 512;
constexpr int LP_MAX_K = 128;
constexpr uint32_t LP_NO_PLACE = 0xFFFFFFFFu;
constexpr float LP_FLOOR = -10000.f;
// Entries of a list that a warp of the gradient looks through by itself.  Of all lists together up to LP_ALONE, and up to 512 a list on average: all, and there is no second kernel (1,000 lists of
// 200 15 us, 18 with it); of a matrix, rows of up to LP_ALONE_ROW, all together LP_ALONE_ALL: with more the registers that this takes tell.
constexpr int LP_LOOK = 1024, LP_ALONE = 1 << 18, LP_ALONE_ROW = 1 << 14, LP_ALONE_ALL = 1 << 21;
// Largest |lse| from which the gradient counts log p: the rounding of lse is an error of every p, of 4e-6 there.
constexpr float LP_NEAR = 64.f;
// Products of the largest score with c up to which d counts from the rounded product: that is half a bit off at most, and 2^d of the largest entry close to 1.
constexpr float LP_SHORT = 16777216.f;

// What a kernel in front may have written: by L2 in a kernel that is launched EARLY, else by L1 (gradient of 1,000 lists of 18,000 51 us, 55 by L2;
// of 600,000 entries and 700 lists of two 97 and 113).
template <bool EARLY, typename T>
__device__ __forceinline__ T lp_get(const T* p) {
    if constexpr (EARLY) return __ldcg(p);
    else return __ldg(p);
}

// Where rows are: a matrix with rows `ld` apart and `cols` long, or lists.  Positions of row r: [begin, end).
struct LpRows {
    const int64_t* offsets;
    int64_t ld, cols, shift, total;  // shift: entries between the boundary and the array; total: entries of all lists
    template <bool EARLY = false>
    __device__ __forceinline__ int64_t begin(int r) const {
        return (offsets ? min(max(lp_get<EARLY>(offsets + r), (int64_t)0), total) : (int64_t)r * ld) + shift;
    }
    template <bool EARLY = false>
    __device__ __forceinline__ int64_t end(int r) const {
        return offsets ? max(min(lp_get<EARLY>(offsets + r + 1), total) + shift, begin<EARLY>(r)) : (int64_t)r * ld + cols + shift;
    }
};

struct LpArgs {
    LpRows rows;
    const int32_t* ids;       // names of the entries of lists, or null
    const int64_t* targets;   // or null
    float* log_probs;         // or null, with targets
    float* entropy;
    float* lse;
    float* top_log_probs;     // or null, with k = 0
    int32_t* top_ids;
    int m, k;
    bool placed;              // log_probs_places_kernel has been launched in front
    float c, inv_t;           // log2(e) / temperature, 1 / temperature
    // rows taken by several CTAs
    int64_t unit;             // positions of a CTA, a multiple of 1,024
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

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float warp_max(float v) {  // NaN where all are
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(r) : "f"(v));
    return r;
}

// A lane's scores of a chunk as they are loaded.  LOW: what -inf counts as, while the largest is above SAFE.
template <typename T>
struct LpRaw;
template <>
struct LpRaw<float> {
    static constexpr float LOW = -1e34f, SAFE = -1e33f;
    alignas(16) float v[LP_PER_LANE<float>];
    __device__ __forceinline__ void put(int j, uint4 w) { *reinterpret_cast<uint4*>(&v[4 * j]) = w; }
    __device__ __forceinline__ void set(int i, float s) { v[i] = s; }
    __device__ __forceinline__ float get(int i) const { return v[i]; }
    __device__ __forceinline__ float top() const {
        float t = fmaxf(v[0], v[1]);
#pragma unroll
        for (int i = 2; i < LP_PER_LANE<float>; ++i) t = fmaxf(t, v[i]);
        return t;
    }
    __device__ __forceinline__ float2 pair(int i) const { return make_float2(max_nan(v[2 * i], LOW), max_nan(v[2 * i + 1], LOW)); }
};
template <typename H>
struct LpRaw16 {
    alignas(16) uint32_t v[LP_PER_LANE<__half> / 2];
    __device__ __forceinline__ void put(int j, uint4 w) { *reinterpret_cast<uint4*>(&v[4 * j]) = w; }
    __device__ __forceinline__ uint32_t half(int i) const { return (i & 1) ? v[i >> 1] >> 16 : v[i >> 1] & 0xFFFFu; }
    __device__ __forceinline__ void put_half(int i, uint32_t h) { v[i >> 1] = (i & 1) ? (v[i >> 1] & 0xFFFFu) | h << 16 : (v[i >> 1] & 0xFFFF0000u) | h; }
};
template <>
struct LpRaw<__nv_bfloat16> : LpRaw16<__nv_bfloat16> {
    static constexpr float LOW = -9.8e33f, SAFE = -1e33f;
    __device__ __forceinline__ void set(int i, float s) { put_half(i, __float_as_uint(s) >> 16); }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(half(i) << 16); }
    __device__ __forceinline__ float top() const {
        uint32_t t = v[0];
#pragma unroll
        for (int i = 1; i < LP_PER_LANE<__half> / 2; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(t) : "r"(v[i]));
        return fmaxf(__uint_as_float(t << 16), __uint_as_float(t & 0xFFFF0000u));
    }
    __device__ __forceinline__ float2 pair(int i) const {
        uint32_t w;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(v[i]), "r"(0xF7F2F7F2u));  // LOW
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
};
template <>
struct LpRaw<__half> : LpRaw16<__half> {
    static constexpr float LOW = -65504.f, SAFE = -40000.f;
    __device__ __forceinline__ void set(int i, float s) { put_half(i, __half_as_ushort(__float2half_rn(s))); }
    __device__ __forceinline__ float get(int i) const { return __half2float(__ushort_as_half((unsigned short)half(i))); }
    __device__ __forceinline__ float top() const {
        uint32_t t = v[0];
#pragma unroll
        for (int i = 1; i < LP_PER_LANE<__half> / 2; ++i) asm("max.f16x2 %0, %0, %1;" : "+r"(t) : "r"(v[i]));
        const float2 f = half_pair(t);
        return fmaxf(f.x, f.y);
    }
    __device__ __forceinline__ float2 pair(int i) const {
        uint32_t w;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(w) : "r"(v[i]), "r"(0xFBFFFBFFu));  // LOW
        return half_pair(w);
    }
};

// Position of a lane's entry i in its chunk.
template <typename T>
__device__ __forceinline__ int lp_place(int lane, int i) {
    constexpr int V = 16 / sizeof(T);
    return ((i / V) * 32 + lane) * V + i % V;
}
// The lane's scores of a chunk, -inf outside [begin, end).  EARLY: in a kernel that is launched early, all of them by L2 (see EightOf; single ones by L1 leave the others eight
// registers: 1,000 x 1M bfloat16 396 us, 440 by L2).  `x`: position 0.
template <bool EARLY, typename T>
__device__ __forceinline__ void lp_load(const T* __restrict__ x, int64_t chunk, int64_t begin, int64_t end, int lane, LpRaw<T>& s) {
    constexpr int V = 16 / sizeof(T);
    const int64_t p0 = chunk * LP_CHUNK<T>;
    if (p0 >= begin && p0 + LP_CHUNK<T> <= end) {
#pragma unroll
        for (int j = 0; j < LP_PER_LANE<T> / V; ++j) s.put(j, __ldcg(reinterpret_cast<const uint4*>(x + p0) + j * 32 + lane));
    } else {
#pragma unroll
        for (int i = 0; i < LP_PER_LANE<T>; ++i) {
            const int64_t p = p0 + lp_place<T>(lane, i);
            s.set(i, p >= begin && p < end ? score_of(EARLY ? __ldcg(x + p) : x[p]) : -INFINITY);
        }
    }
}

// A warp's chunks first, first + step, ... below last, all in one row; `leave(chunk, top)` takes the chunks' maxima, `largest` becomes the
// lane's.  The next chunk is on its way while one is summed.
template <bool EARLY, typename T, typename Leave>
__device__ __forceinline__ LpPart lp_chunks(const T* __restrict__ x, int64_t first, int64_t last, int step, int64_t begin, int64_t end, float c, int lane,
                                            float& largest, Leave leave) {
    float m = LpPart::none().m, mc = __fmul_rn(m, c);  // the same in all lanes; mc: what d counts from in the short way, rounded wherever it is used
    const bool common = c > 0.01f && c < 1e4f;
    auto is_short = [&](float m, float mc) { return common && m > LpRaw<T>::SAFE && fabsf(mc) < LP_SHORT; };
    auto in_short = [&]() { return is_short(m, mc); };
    float2 l = make_float2(0.f, 0.f), e = l;
    LpRaw<T> next;
    if (first < last) lp_load<EARLY>(x, first, begin, end, lane, next);
#pragma unroll 1
    for (int64_t chunk = first; chunk < last; chunk += step) {
        const LpRaw<T> s = next;
        if (chunk + step < last) lp_load<EARLY>(x, chunk + step, begin, end, lane, next);
        float top = s.top();
        largest = fmaxf(largest, top);
        top = warp_max(top);
        if (top != top) top = -INFINITY;
        leave(chunk, top);
        if (top > m) {
            const float to = __fmul_rn(top, c);
            const bool was = in_short(), is = is_short(top, to);
            // from what the sums are relative to, mc or m c itself, to what they will be
            const float d = max_nan(was ? (is ? mc - to : -fmaf(top, c, -mc)) : is ? fmaf(m, c, -to) : (m - top) * c, LP_FLOOR), f = exp2_fast(d);
            e.x = (e.x + l.x * d) * f;
            e.y = (e.y + l.y * d) * f;
            l.x *= f;
            l.y *= f;
            m = top;
            mc = to;
        }
        if (in_short()) {
            const float2 c2 = make_float2(c, c), from = make_float2(-mc, -mc);
            float2 lc = make_float2(0.f, 0.f), ec = lc;  // of the chunk: thousands of terms one by one into one sum cost it two digits
#pragma unroll
            for (int i = 0; i < LP_PER_LANE<T> / 2; ++i) {
                const float2 d = fma2(s.pair(i), c2, from), p = make_float2(exp2_fast(d.x), exp2_fast(d.y));
                lc = add2(lc, p);
                ec = fma2(p, d, ec);
            }
            l = add2(l, lc);
            e = add2(e, ec);
        } else {
#pragma unroll
            for (int i = 0; i < LP_PER_LANE<T>; ++i) {
                const float d = max_nan((s.get(i) - m) * c, LP_FLOOR), p = exp2_fast(d);
                l.x += p;
                e.x = fmaf(p, d, e.x);
            }
        }
    }
    LpPart part{m, l.x + l.y, e.x + e.y};
    const float off = in_short() ? fmaf(m, c, -mc) : 0.f, f = exp2_fast(-off);  // from mc to m itself
    part.e = (part.e - off * part.l) * f;
    part.l *= f;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        part.l += __shfl_xor_sync(0xFFFFFFFFu, part.l, o);
        part.e += __shfl_xor_sync(0xFFFFFFFFu, part.e, o);
    }
    return part;
}

// What a CTA of TH threads shares.
template <int TH>
struct LpShared {
    static constexpr int CHUNKS = 4 * TH;     // maxima that a CTA keeps of a row; a longer row's stand for several chunks each
    static constexpr int STEP = 4 * TH;       // entries that are looked at before the collected ones are counted
    static constexpr int KEYS = STEP + (STEP > LP_MAX_K ? STEP : LP_MAX_K);
    uint64_t keys[KEYS];
    uint32_t maxima[CHUNKS];
    LpPart parts[TH / 32];
    int count;
    int64_t target;  // position of the given entry, or -1
};

// The CTA's part from its warps', in the order of the warps; for all threads.
template <int TH>
__device__ __forceinline__ LpPart lp_join_warps(LpShared<TH>& sh, const LpPart& mine, float c) {
    if ((threadIdx.x & 31) == 0) sh.parts[threadIdx.x >> 5] = mine;
    __syncthreads();
    LpPart all = sh.parts[0];
#pragma unroll
    for (int w = 1; w < TH / 32; ++w) all.join(sh.parts[w], c);
    return all;
}

// Sorts keys[0, n), n a power of two, the largest first.
template <int TH>
__device__ __forceinline__ void lp_sort(uint64_t* keys, int n) {
    for (int size = 2; size <= n; size *= 2) {
        for (int stride = size / 2; stride; stride >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += TH) {
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
template <int TH>
__device__ __forceinline__ void lp_settle(LpShared<TH>& sh, int k) {
    __syncthreads();
    const int count = sh.count;
    int n = 2;
    while (n < count) n *= 2;
    for (int i = count + threadIdx.x; i < n; i += TH) sh.keys[i] = 0;
    lp_sort<TH>(sh.keys, n);
    if (threadIdx.x == 0) sh.count = min(count, k);
    __syncthreads();
}
// The k largest keys of key(0 .. n - 1) that are at least `least`, sorted, into sh.keys; sh.count of them.  Keys differ from one another, 0 is none.
template <int TH, typename Key>
__device__ __forceinline__ void lp_largest(LpShared<TH>& sh, int64_t n, int k, uint64_t least, Key key) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int64_t i0 = 0; i0 < n; i0 += LpShared<TH>::STEP) {
        uint64_t v[LpShared<TH>::STEP / TH];
#pragma unroll
        for (int j = 0; j < LpShared<TH>::STEP / TH; ++j) {
            const int64_t i = i0 + j * TH + threadIdx.x;
            v[j] = i < n ? key(i) : 0ull;
        }
#pragma unroll
        for (int j = 0; j < LpShared<TH>::STEP / TH; ++j)
            if (v[j] && v[j] >= least) sh.keys[atomicAdd(&sh.count, 1)] = v[j];
        __syncthreads();
        if (sh.count > LpShared<TH>::KEYS - LpShared<TH>::STEP) {
            lp_settle(sh, k);
            if (sh.count == k) least = max(least, sh.keys[k - 1]);
        }
        __syncthreads();
    }
    lp_settle(sh, k);
}
// The k-th largest of the threads' scores, k <= TH.
template <int TH>
__device__ __forceinline__ float lp_bound(LpShared<TH>& sh, float mine, int k) {
    __syncthreads();
    sh.keys[threadIdx.x] = lp_order(mine);
    lp_sort<TH>(sh.keys, TH);
    const float bound = lp_score((uint32_t)sh.keys[k - 1]);
    __syncthreads();
    return bound;
}

// Position of the entry that a target names in a row, or -1 where it does not stand where ascending ids would have it; by one warp.  The first 32 ids that it looks at (all, where there
// are no more) can be asked for long before.
template <bool EARLY = false>
struct LpFind {
    int64_t lo, hi, step, target;  // ids below lo are smaller, at and behind hi larger
    int32_t id;
    __device__ __forceinline__ void probe(const int32_t* __restrict__ ids) {
        step = (hi - lo + 31) / 32;
        const int64_t p = lo + (threadIdx.x & 31) * step;
        id = p < hi ? lp_get<EARLY>(ids + p) : 0x7FFFFFFF;
    }
    __device__ __forceinline__ LpFind(const LpArgs& a, int row, int64_t begin, int64_t end) : lo(begin), hi(end), step(1), target(lp_get<EARLY>(a.targets + row)), id(0) {
        if (a.ids && hi > lo) probe(a.ids - a.rows.shift);
    }
    __device__ __forceinline__ int64_t operator()(const LpArgs& a) {
        if (!a.ids) return target >= 0 && target < hi - lo ? lo + target : -1;
        const int lane = threadIdx.x & 31;
        while (hi > lo) {
            const bool in = lo + lane * step < hi;
            const unsigned smaller = __ballot_sync(0xFFFFFFFFu, in && id < target), same = __ballot_sync(0xFFFFFFFFu, in && id == target);
            if (same) return lo + (int64_t)(__ffs((int)same) - 1) * step;
            const int n = __popc(smaller);  // the first n probes
            if (!n) return -1;
            hi = min(hi, lo + n * step);
            lo = lo + (n - 1) * step + 1;
            if (hi > lo) probe(a.ids - a.rows.shift);
        }
        return -1;
    }
};

// The first entry of [begin, end) that a target names, of those that thread `thread` of `threads` looks at, or `end`.  For lists in any order: that the search does not find an id says nothing
// of them.  N loads of a thread are on their way at a time.
template <int N>
__device__ __forceinline__ int64_t lp_first_named(const int32_t* __restrict__ names, int64_t begin, int64_t end, int64_t target, int thread, int threads) {
    const int32_t name = (int32_t)target;
    if (name != target) return end;
#pragma unroll 1
    for (int64_t p0 = begin - (int64_t)((uintptr_t)(names + begin) / 4 % 4) + 4 * thread; p0 < end; p0 += (int64_t)4 * N * threads) {
        int4 w[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t p = p0 + (int64_t)4 * j * threads;
            if (p >= begin && p + 4 <= end) {
                w[j] = __ldcg(reinterpret_cast<const int4*>(names + p));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) reinterpret_cast<int32_t*>(&w[j])[i] = p + i >= begin && p + i < end ? __ldcg(names + p + i) : ~name;
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = w[j].x == name ? 0 : w[j].y == name ? 1 : w[j].z == name ? 2 : w[j].w == name ? 3 : -1;
            if (at >= 0) return p0 + (int64_t)4 * j * threads + at;
        }
    }
    return end;
}
// By a CTA whose threads have seen that `found`, in shared memory, is -1: the first entry of the row, if there is one.
template <int N = 4>
__device__ __forceinline__ void lp_find_in_any_order(const LpArgs& a, int row, int64_t begin, int64_t end, int64_t& found, int threads) {
    const int64_t first = lp_first_named<N>(a.ids - a.rows.shift, begin, end, __ldcg(a.targets + row), threadIdx.x, threads);
    __syncthreads();
    if (first < end) atomicMin(reinterpret_cast<unsigned long long*>(&found), (unsigned long long)first);
    __syncthreads();
}
// Whether a list can have an entry that the search did not find.
__device__ __forceinline__ bool lp_may_be_left(int64_t begin, int64_t end) { return end - begin > 32; }

// Lists [0, m) by CTAs of LP_WARPS warps, of which this is the one `cta` of `ctas`: look(row) by a warp for those that may(row) says so of, then rest(row) by the CTA where that was true.
template <typename May, typename Look, typename Rest>
__device__ __forceinline__ void lp_by_warps_then_ctas(int m, int cta, int ctas, May may, Look look, Rest rest) {
    __shared__ unsigned s_left[LP_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = min((m - 1) / (ctas * LP_WARPS) + 1, 32);  // lists for a warp at a time
    for (int64_t row0 = (int64_t)cta * LP_WARPS * per; row0 < m; row0 += (int64_t)ctas * LP_WARPS * per) {
        const int64_t mine = row0 + warp * per + lane;
        unsigned left = 0;
        for (unsigned some = __ballot_sync(0xFFFFFFFFu, lane < per && mine < m && may((int)mine)); some; some &= some - 1)
            if (look((int)(row0 + warp * per) + __ffs((int)some) - 1)) left |= some & -some;
        if (lane == 0) s_left[warp] = left;
        __syncthreads();
        for (int w = 0; w < LP_WARPS; ++w)
            for (unsigned some = s_left[w]; some; some &= some - 1) rest((int)(row0 + w * per) + __ffs((int)some) - 1);
        __syncthreads();
    }
}

// What a row's result is made of, by the whole CTA.  `maximum`: orders of the largest scores of groups of 1 << wide chunks from first_chunk on; `largest`: a thread's own score, of no
// other's entry.
template <int TH, bool EARLY, typename T, typename Maximum>
__device__ __forceinline__ void lp_finish(const T* __restrict__ x, const LpArgs& a, LpShared<TH>& sh, int row, int64_t begin, int64_t end, LpPart all,
                                          Maximum maximum, int64_t first_chunk, int64_t last_chunk, int wide, float largest) {
    if (a.targets && a.ids) {
        if (a.placed) {
            asm volatile("griddepcontrol.wait;" ::: "memory");  // for log_probs_places_kernel
            if (threadIdx.x == 0) {  // who needs it and overwrites it
                const uint32_t place = __ldcg(reinterpret_cast<const uint32_t*>(a.log_probs) + row);
                sh.target = place == LP_NO_PLACE ? -1 : begin + place;
            }
        } else if (sh.target < 0 && lp_may_be_left(begin, end)) {
            lp_find_in_any_order(a, row, begin, end, sh.target, TH);
        }
    }
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
        if (a.targets) a.log_probs[row] = sh.target < 0 ? -INFINITY : log_p(score_of(__ldcg(x + sh.target)));
    }
    if (!a.k) return;
    const float bound = lp_bound(sh, largest, a.k);
    const uint32_t least = max(lp_order(bound), 0x00800000u);  // more than -inf
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t c0 = first_chunk + warp * 32; c0 < last_chunk; c0 += TH) {  // a lane looks at a chunk's maximum
        const int64_t mine = c0 + lane;
        unsigned reach = __ballot_sync(0xFFFFFFFFu, mine < last_chunk && maximum((mine - first_chunk) >> wide) >= least);
        for (; reach; reach &= reach - 1) {
            const int64_t chunk = c0 + __ffs((int)reach) - 1;
            LpRaw<T> s;
            lp_load<EARLY>(x, chunk, begin, end, lane, s);
            if (!(s.top() >= bound)) continue;
#pragma unroll
            for (int j = 0; j < LP_PER_LANE<T>; ++j) {
                const float v = s.get(j);
                if (v >= bound && v > -INFINITY) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < LpShared<TH>::KEYS) sh.keys[at] = (uint64_t)lp_order(v) << 32 | (0xFFFFFFFFu - (uint32_t)(chunk * LP_CHUNK<T> + lp_place<T>(lane, j) - begin));
                }
            }
        }
    }
    __syncthreads();
    if (sh.count <= LpShared<TH>::KEYS) {
        lp_settle(sh, a.k);
    } else {  // many that are alike
        lp_largest(sh, end - begin, a.k, (uint64_t)least << 32, [&](int64_t i) {
            const float v = score_of(__ldcg(x + begin + i));
            return v > -INFINITY ? (unsigned long long)lp_order(v) << 32 | (0xFFFFFFFFu - (uint32_t)i) : 0ull;
        });
    }
    for (int i = threadIdx.x; i < a.k; i += TH) {
        float lp = -INFINITY;
        int32_t id = -1;
        if (i < sh.count) {
            const uint32_t at = 0xFFFFFFFFu - (uint32_t)sh.keys[i];
            const float s = lp_score((uint32_t)(sh.keys[i] >> 32));
            if (s * a.inv_t > -INFINITY) {
                lp = log_p(s);
                id = a.ids ? __ldcg(a.ids - a.rows.shift + begin + at) : (int32_t)at;
            }
        }
        a.top_log_probs[(int64_t)row * a.k + i] = lp;
        a.top_ids[(int64_t)row * a.k + i] = id;
    }
}

// Long lists: where the entries are that targets name, before the pass needs to know.  A list whose target is not where a search finds it is looked through, for which a CTA of the pass may be a
// warp: that warp's list took twice as long, and was the last (10,000 lists of 18,000 float32, a tenth of the targets in none: 324 us, 210 without looking through).  Places in the
// list wait in the row's log probability until the pass puts that there.
__global__ void __launch_bounds__(LP_THREADS) log_probs_places_kernel(LpArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ int64_t s_found;
    uint32_t* const places = reinterpret_cast<uint32_t*>(a.log_probs);
    lp_by_warps_then_ctas(
        a.m, blockIdx.x, gridDim.x, [](int) { return true; },
        [&](int row) {
            const int64_t begin = a.rows.begin(row), end = a.rows.end(row), at = LpFind<>(a, row, begin, end)(a);
            if ((threadIdx.x & 31) == 0) places[row] = at < 0 ? LP_NO_PLACE : (uint32_t)(at - begin);
            return at < 0 && lp_may_be_left(begin, end);
        },
        [&](int row) {
            const int64_t begin = a.rows.begin(row), end = a.rows.end(row);
            if (threadIdx.x == 0) s_found = -1;
            lp_find_in_any_order<8>(a, row, begin, end, s_found, LP_THREADS);
            if (threadIdx.x == 0 && s_found >= 0) places[row] = (uint32_t)(s_found - begin);
            __syncthreads();
        });
}

// A CTA of TH threads for each row.
template <int TH, typename T>
__global__ void __launch_bounds__(TH) log_probs_row_kernel(const T* __restrict__ x, LpArgs a) {
    __shared__ LpShared<TH> sh;
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t begin = a.rows.begin(row), end = a.rows.end(row);
    const int64_t first = begin / LP_CHUNK<T>, last = end > begin ? (end + LP_CHUNK<T> - 1) / LP_CHUNK<T> : first;
    int wide = 0;
    while ((last - first + (1ll << wide) - 1) >> wide > LpShared<TH>::CHUNKS) ++wide;
    const int groups = (int)((last - first + (1ll << wide) - 1) >> wide);
    if (a.k) {
        for (int i = threadIdx.x; i < groups; i += TH) sh.maxima[i] = 0;
        __syncthreads();
    }
    auto leave = [&](int64_t chunk, float top) {
        if (a.k && lane == 0) atomicMax(&sh.maxima[(chunk - first) >> wide], lp_order(top));
    };
    LpPart mine;
    float largest = -INFINITY;
    if (warp == TH / 32 - 1 && a.targets && !a.placed) {  // the warp with the fewest chunks
        LpFind<> find(a, row, begin, end);
        mine = lp_chunks<false>(x, first + warp, last, TH / 32, begin, end, a.c, lane, largest, leave);
        const int64_t at = find(a);
        if (lane == 0) sh.target = at;
    } else {
        mine = lp_chunks<false>(x, first + warp, last, TH / 32, begin, end, a.c, lane, largest, leave);
    }
    const LpPart all = lp_join_warps(sh, mine, a.c);
    lp_finish<TH, false>(x, a, sh, row, begin, end, all, [&](int64_t i) { return sh.maxima[i]; }, first, last, wide, largest);
}

// Rows taken by several CTAs.  Slots of a row's units and chunks: blocks of `size` positions from the one that it begins in on; lists share the numbering of all
// positions, moved on by one for each list, so that no two share a slot.
__device__ __forceinline__ int64_t lp_slot(const LpArgs& a, int row, int64_t begin, int64_t size, int64_t per_row) {
    return a.rows.offsets ? begin / size + row : (int64_t)row * per_row;
}
template <typename T>
__device__ __forceinline__ int64_t lp_chunks_per_row(const LpArgs& a) { return a.rows.cols / LP_CHUNK<T> + 2; }

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_unit_kernel(const T* __restrict__ x, LpArgs a, KernelBefore before) {
    behind_kernel_before(x, before);
    __shared__ LpShared<LP_THREADS> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int row;
    int64_t nth;
    if (a.rows.offsets) {  // the last list whose first slot is not behind this one
        int lo = 0, hi = a.m;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (lp_slot(a, mid, a.rows.begin<true>(mid), a.unit, 0) <= (int64_t)blockIdx.x) lo = mid;
            else hi = mid;
        }
        row = lo;
        nth = (int64_t)blockIdx.x - lp_slot(a, row, a.rows.begin<true>(row), a.unit, 0);
    } else {
        row = (int)(blockIdx.x / (unsigned)a.units_per_row);
        nth = blockIdx.x - (unsigned)row * (unsigned)a.units_per_row;
    }
    const int64_t begin = a.rows.begin<true>(row), end = a.rows.end<true>(row);
    const int64_t from = max((begin / a.unit + nth) * a.unit, begin), to = min((begin / a.unit + nth + 1) * a.unit, end);
    if (from >= to) return;
    const int64_t slot = lp_slot(a, row, begin, LP_CHUNK<T>, lp_chunks_per_row<T>(a)), first = begin / LP_CHUNK<T>;
    float largest = -INFINITY;
    const LpPart mine = lp_chunks<true>(x, from / LP_CHUNK<T> + warp, (to + LP_CHUNK<T> - 1) / LP_CHUNK<T>, LP_WARPS, begin, end, a.c, lane, largest, [&](int64_t chunk, float top) {
        if (a.k && lane == 0) a.maxima[slot + chunk - first] = lp_order(top);
    });
    const LpPart all = lp_join_warps(sh, mine, a.c);
    if (threadIdx.x == 0) a.parts[blockIdx.x] = make_float4(all.m, all.l, all.e, 0.f);
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_join_kernel(const T* __restrict__ x, LpArgs a, KernelBefore before) {
    behind_kernel_before(x, before);
    __shared__ LpShared<LP_THREADS> sh;
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t begin = a.rows.begin<true>(row), end = a.rows.end<true>(row);
    if (warp == 0 && a.targets) {
        const int64_t at = LpFind<true>(a, row, begin, end)(a);
        if (lane == 0) sh.target = at;
    }
    const int64_t units = end > begin ? (end - 1) / a.unit - begin / a.unit + 1 : 0, slot = lp_slot(a, row, begin, a.unit, a.units_per_row);
    LpPart mine = LpPart::none();
    for (int64_t u = threadIdx.x; u < units; u += LP_THREADS) {
        const float4 p = __ldcg(a.parts + slot + u);
        mine.join(LpPart{p.x, p.y, p.z}, a.c);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mine.join(mine.shuffled(o), a.c);
    const LpPart all = lp_join_warps(sh, mine, a.c);
    const int64_t first = begin / LP_CHUNK<T>, last = end > begin ? (end + LP_CHUNK<T> - 1) / LP_CHUNK<T> : first;
    const uint32_t* const maxima = a.maxima + lp_slot(a, row, begin, LP_CHUNK<T>, lp_chunks_per_row<T>(a));
    auto maximum = [&](int64_t i) { return __ldcg(maxima + i); };
    float largest = -INFINITY;
    if (a.k && last - first >= LP_THREADS) {  // of every 256th chunk
        for (int64_t c = threadIdx.x; c < last - first; c += LP_THREADS) largest = fmaxf(largest, lp_score(max(maximum(c), 0x007FFFFFu)));
    } else if (a.k) {  // too few: of every eighth chunk's entries of a lane
        for (int64_t c = first + warp; c < last; c += LP_WARPS) {
            LpRaw<T> s;
            lp_load<true>(x, c, begin, end, lane, s);
            largest = fmaxf(largest, s.top());
        }
    }
    lp_finish<LP_THREADS, true>(x, a, sh, row, begin, end, all, maximum, first, last, 0, largest);
}

// ------------------------------------------------------------------------------------------
// Gradient.  Bound by HBM and issue (59 and 74 %): 1,000 x 200,003 bfloat16 151 us (5.3 TB/s, half of it written), float32 266 (6.0); rows of scores and gradient that begin differently 300 and 361.  Two loads of a thread
// in flight and six CTAs an SM: four loads and the four CTAs that they leave room for took 174 and 289.
// ------------------------------------------------------------------------------------------
struct LpBackward {
    LpArgs f;
    const float* lse;
    const float* entropy;
    const float* g;         // of the log probabilities, or null
    const float* h;         // of the entropies, or null
    int64_t ldo;            // of the result, where it is a matrix
    int64_t units;          // spans of positions: of all lists, or that a matrix's row can reach into
    int span;               // positions of lists for a warp
    int whole, shares;      // CTAs of log_probs_backward_whole_kernel, and how many of them have a row
};

// Constants of a row: ds = p (a - b log p), and more at the given entry; log p = z - lse, a = own - g, own = -h entropy / temperature, b = h / temperature, g by the temperature.
struct LpRowTerms {
    float lse, a, b, g, own;
    float base;  // log p = (s - base) / temperature - lse where a row is taken as a whole; else 0, and not used
    int64_t target;
    bool bad;    // lse is NaN: so is everything but what is masked
};

template <typename T>
__device__ __forceinline__ LpRowTerms lp_row_terms(const T* __restrict__ x, const LpBackward& b, int row, int64_t target) {
    LpRowTerms r;
    const float h = b.h ? __ldg(b.h + row) : 0.f, entropy = __ldg(b.entropy + row);
    float g = b.f.targets && b.g ? __ldg(b.g + row) : 0.f;
    r.lse = __ldg(b.lse + row);
    if (r.lse == -INFINITY) r.lse = 0.f;  // all masked: 2^-inf is 0 then
    r.bad = r.lse != r.lse;
    r.base = 0.f;
    r.target = target;
    if (target < 0 || score_of(x[target]) * b.f.inv_t == -INFINITY) {  // a log probability of -inf stays where it is
        r.target = -1;
        g = 0.f;
    }
    r.own = -(h * entropy) * b.f.inv_t;
    r.b = h * b.f.inv_t;
    r.g = g * b.f.inv_t;
    r.a = r.own - r.g;
    return r;
}
__device__ __forceinline__ bool lp_far(const LpBackward& b, int row) {
    const float lse = __ldg(b.lse + row);
    return fabsf(lse) > LP_NEAR && lse != -INFINITY;
}
// Where the lse that is given is that of these scores but for its rounding, log p counts from the largest score.
__device__ __forceinline__ void lp_count_from_largest(LpRowTerms& r, const LpPart& all, float inv_t) {
    const float log_l = logf(all.l), lse = all.m * inv_t + log_l;
    if (all.l > 0.f && (lse == r.lse || fabsf(lse - r.lse) <= 4.8e-7f * fabsf(lse))) {
        r.base = all.m;
        r.lse = log_l;
    }
}
// The entry that has the gradient of a row's log probability, or -1; by a warp.  `left`: of a list of more than `look` entries, whose target is not where the search finds it, if it has it.
__device__ __forceinline__ int64_t lp_given(const LpBackward& b, int row, int64_t begin, int64_t end, int64_t look, bool& left) {
    left = false;
    if (!b.f.targets || !b.g) return -1;
    int64_t at = LpFind<>(b.f, row, begin, end)(b.f);
    if (at < 0 && b.f.ids && lp_may_be_left(begin, end)) {
        left = end - begin > look;
        if (!left) {
            at = lp_first_named<2>(b.f.ids - b.f.rows.shift, begin, end, __ldg(b.f.targets + row), threadIdx.x & 31, 32);
            const unsigned first = __reduce_min_sync(0xFFFFFFFFu, (unsigned)(at - begin));  // 32 bits are enough for the lists that are looked through here
            at = first < (unsigned)(end - begin) ? begin + first : -1;
        }
    }
    return at;
}
template <bool WHOLE>
__device__ __forceinline__ float2 lp_grad(const LpRowTerms& r, float2 s, float inv_t) {
    if constexpr (WHOLE) s = make_float2(s.x - r.base, s.y - r.base);
    float2 lp = fma2(s, make_float2(inv_t, inv_t), make_float2(-r.lse, -r.lse));
    lp = make_float2(max_nan(lp.x, LP_FLOOR), max_nan(lp.y, LP_FLOOR));  // no 0 times infinity for what is masked, or as low as that
    const float2 q = mul2(lp, make_float2(1.4426950409f, 1.4426950409f));
    float2 v = mul2(make_float2(exp2_fast(q.x), exp2_fast(q.y)), fma2(make_float2(-r.b, -r.b), lp, make_float2(r.a, r.a)));
    if (r.bad) v = make_float2(s.x == -INFINITY ? 0.f : v.x, s.y == -INFINITY ? 0.f : v.y);
    return v;
}
// At the given entry.  1 - p of one that is nearly certain is as exact as its log p: lists of one or two entries have hardly anything else; nor may a large g take the entropy's part with it.
template <bool WHOLE>
__device__ __forceinline__ float lp_grad_given(const LpRowTerms& r, float s, float inv_t) {
    if constexpr (WHOLE) s -= r.base;
    const float lp = max_nan(fmaf(s, inv_t, -r.lse), LP_FLOOR), p = exp2_fast(lp * 1.4426950409f);
    return fmaf(p, fmaf(-r.b, lp, r.own), -r.g * expm1f(lp));
}
__device__ __forceinline__ void put_grad(float* o, float v) { *o = v; }
__device__ __forceinline__ void put_grad(__half* o, float v) { *o = __float2half_rn(v); }
__device__ __forceinline__ void put_grad(__nv_bfloat16* o, float v) { *o = __float2bfloat16_rn(v); }

// Positions [from, to) of a row by `threads` threads, whose `thread` this is, 32 bytes of each in flight; `x` and `o`: position 0 of the scores, on a 16-byte boundary, and of the gradient.
// ALIKE: that is on a boundary, too, in every row.
template <bool ALIKE, bool WHOLE, typename T>
__device__ __forceinline__ void lp_backward_span(const T* __restrict__ x, T* __restrict__ o, const LpRowTerms& r, float inv_t, int64_t from, int64_t to, int thread,
                                                 int threads) {
    constexpr int V = 16 / sizeof(T);
    if constexpr (!ALIKE) {  // an entry at a time, sixteen of them on their way
#pragma unroll 1
        for (int64_t p0 = from + thread; p0 < to; p0 += (int64_t)16 * threads) {
            float s[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = p0 + (int64_t)i * threads < to ? score_of(x[p0 + (int64_t)i * threads]) : 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float2 d = lp_grad<WHOLE>(r, make_float2(s[i], s[i + 1]), inv_t);
                const int64_t p = p0 + (int64_t)i * threads, p1 = p + threads;
                if (p < to) put_grad(o + p, p == r.target ? lp_grad_given<WHOLE>(r, s[i], inv_t) : d.x);
                if (p1 < to) put_grad(o + p1, p1 == r.target ? lp_grad_given<WHOLE>(r, s[i + 1], inv_t) : d.y);
            }
        }
    } else {
        for (int64_t p0 = from / V * V + (int64_t)thread * V; p0 < to; p0 += (int64_t)2 * threads * V) {
            uint4 w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t p = p0 + (int64_t)j * threads * V;
                if (p >= from && p + V <= to) {
                    w[j] = __ldg(reinterpret_cast<const uint4*>(x + p));
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) reinterpret_cast<T*>(&w[j])[i] = p + i >= from && p + i < to ? x[p + i] : T(0.f);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t p = p0 + (int64_t)j * threads * V;
                if (p >= to) break;
                float v[V];
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const T* const t = reinterpret_cast<const T*>(&w[j]) + i;
                    const float2 d = lp_grad<WHOLE>(r, make_float2(score_of(t[0]), score_of(t[1])), inv_t);
                    v[i] = d.x;
                    v[i + 1] = d.y;
                }
                if (r.target >= p && r.target < p + V) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (p + i == r.target) v[i] = lp_grad_given<WHOLE>(r, score_of(reinterpret_cast<const T*>(&w[j])[i]), inv_t);
                }
                if (p >= from && p + V <= to) {
                    uint4 u;
                    if constexpr (sizeof(T) == 4) {
                        u = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                    } else {
                        u = make_uint4(pack_scores(o, v[0], v[1]), pack_scores(o, v[2], v[3]), pack_scores(o, v[4], v[5]), pack_scores(o, v[6], v[7]));
                    }
                    *reinterpret_cast<uint4*>(o + p) = u;
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (p + i >= from && p + i < to) put_grad(o + p + i, v[i]);
                }
            }
        }
    }
}

// Largest score and sums of a row, by a CTA.
template <typename T>
__device__ __forceinline__ LpPart lp_part_by_cta(const T* __restrict__ x, const LpBackward& b, int64_t begin, int64_t end, LpPart* s_parts) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float largest = 0.f;
    const LpPart mine = lp_chunks<false>(x, begin / LP_CHUNK<T> + warp, (end + LP_CHUNK<T> - 1) / LP_CHUNK<T>, LP_WARPS, begin, end, b.f.c, lane, largest, [](int64_t, float) {});
    if (lane == 0) s_parts[warp] = mine;
    __syncthreads();
    LpPart all = s_parts[0];
    for (int w = 1; w < LP_WARPS; ++w) all.join(s_parts[w], b.f.c);
    return all;
}

// A CTA for a span of a matrix's row.
template <typename T>
constexpr int LP_ROW_SPAN = 4 * LP_THREADS * (16 / sizeof(T));
// ALONE: of short rows.  What a row that log_probs_backward_whole_kernel is there for needs to be looked at for, each span's CTA looks at by itself.
template <bool ALIKE, bool ALONE, typename T>
__global__ void __launch_bounds__(LP_THREADS, ALONE ? 3 : ALIKE ? 6 : 4) log_probs_backward_rows_kernel(const T* __restrict__ x, T* __restrict__ out, LpBackward b) {
    const int64_t row = blockIdx.x / (unsigned)b.units, begin = b.f.rows.begin((int)row), end = b.f.rows.end((int)row);
    const int64_t span = begin / LP_ROW_SPAN<T> + (blockIdx.x - (unsigned)row * (unsigned)b.units);
    const int64_t from = max(span * LP_ROW_SPAN<T>, begin), to = min((span + 1) * LP_ROW_SPAN<T>, end);
    const bool far = lp_far(b, (int)row);
    if (from < to && (ALONE || !far)) {
        bool left;
        LpRowTerms r = lp_row_terms(x, b, (int)row, lp_given(b, (int)row, begin, end, LP_LOOK, left));
        if constexpr (ALONE) {
            if (far) {
                __shared__ LpPart s_parts[LP_WARPS];
                lp_count_from_largest(r, lp_part_by_cta(x, b, begin, end, s_parts), b.f.inv_t);
            }
        }
        lp_backward_span<ALIKE, ALONE>(x, out + (row * b.ldo - begin), r, b.f.inv_t, from, to, threadIdx.x, LP_THREADS);
    }
    if (!ALONE && blockIdx.x + 1 == gridDim.x) asm volatile("griddepcontrol.wait;" ::: "memory");  // what comes next waits for log_probs_backward_whole_kernel, too
}

// A warp for a span of all lists' positions, and for each list in it: what it has to know of a list takes longer than a short one.
template <bool ALIKE, bool ALONE, typename T>
__global__ void __launch_bounds__(LP_THREADS, ALONE ? 3 : ALIKE ? 6 : 4) log_probs_backward_lists_kernel(const T* __restrict__ x, T* __restrict__ out, LpBackward b) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t n = (int64_t)blockIdx.x * LP_WARPS + (threadIdx.x >> 5);
    if (n >= b.units) return;
    const LpRows& rows = b.f.rows;
    const int64_t p0 = n * b.span, p1 = p0 + b.span;
    for (int row = owner_of(rows.offsets, b.f.m, max(p0 - rows.shift, (int64_t)0)); row < b.f.m; ++row) {
        const int64_t begin = rows.begin(row), end = rows.end(row);
        if (begin >= p1) break;
        const int64_t from = max(begin, p0), to = min(end, p1);
        if (from >= to) continue;
        const bool far = lp_far(b, row);
        if (!ALONE && far) continue;
        bool left;  // then as if it had no target; log_probs_backward_whole_kernel looks for that
        LpRowTerms r = lp_row_terms(x, b, row, lp_given(b, row, begin, end, ALONE ? LP_ALONE : LP_LOOK, left));
        if constexpr (ALONE) {
            if (far) {
                float largest = 0.f;
                const LpPart all = lp_chunks<false>(x, begin / LP_CHUNK<T>, (end + LP_CHUNK<T> - 1) / LP_CHUNK<T>, 1, begin, end, b.f.c, threadIdx.x & 31, largest, [](int64_t, float) {});
                lp_count_from_largest(r, all, b.f.inv_t);
            }
        }
        lp_backward_span<ALIKE, ALONE>(x, out - rows.shift, r, b.f.inv_t, from, to, threadIdx.x & 31, 32);
    }
}

// Rows that have to be looked at as a whole, beside the kernel of the spans.  Rows whose lse is large, so that it says p only to its rounding (squared distances of bytes by a temperature of
// 0.05: to 10 %), are left to this one: their log p counts from the largest score, as in the forward pass, with sums made again (1,000 x 200,003 bfloat16, all of them such rows, 450 us in place
// of 157).  Long lists whose target is not where a search finds it are looked through; where it is found after all, the kernel of the spans is waited for and the list is done again.
// (As CTAs of its launch this took registers from the spans: 186 us in place of 157.)  Beside the spans of a matrix it is launched first, which is sooner, beside those of lists behind them.
template <bool ALIKE, typename T>
__global__ void __launch_bounds__(LP_THREADS, 4) log_probs_backward_whole_kernel(const T* __restrict__ x, T* __restrict__ out, LpBackward b) {
    __shared__ int64_t s_target;
    __shared__ LpPart s_parts[LP_WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a matrix's spans
    const LpRows& rows = b.f.rows;
    // few rows have several CTAs each, which look through all of it and take their share of what follows
    const int share = (int)blockIdx.x % b.shares;
    lp_by_warps_then_ctas(
        b.f.m, (int)blockIdx.x / b.shares, b.whole / b.shares,
        [&](int row) { return (b.f.ids && b.g && rows.end(row) - rows.begin(row) > LP_LOOK) || lp_far(b, row); },
        [&](int row) {
            bool left = lp_far(b, row);
            if (!left) lp_given(b, row, rows.begin(row), rows.end(row), LP_LOOK, left);
            return left;
        },
        [&](int row) {
            const int64_t begin = rows.begin(row), end = rows.end(row);
            if (threadIdx.x == 0) s_target = -1;
            __syncthreads();
            const bool far = lp_far(b, row);
            if (b.f.targets && b.g) {
                const int64_t at = far ? LpFind<>(b.f, row, begin, end)(b.f) : -1;  // the same in all warps; of the others it is known
                if (at < 0 && b.f.ids && lp_may_be_left(begin, end)) lp_find_in_any_order<8>(b.f, row, begin, end, s_target, LP_THREADS);
                else if (threadIdx.x == 0) s_target = at;
            }
            __syncthreads();
            if (!far) {
                if (s_target < 0) {  // it has none, as has been taken for granted
                    __syncthreads();
                    return;
                }
                asm volatile("griddepcontrol.wait;" ::: "memory");  // for the spans of lists
            }
            LpRowTerms r = lp_row_terms(x, b, row, s_target);
            if (far) lp_count_from_largest(r, lp_part_by_cta(x, b, begin, end, s_parts), b.f.inv_t);
            const int64_t each = ((end - begin) / b.shares / 16 + 1) * 16, from = begin + share * each;
            lp_backward_span<ALIKE, true>(x, rows.offsets ? out - rows.shift : out + ((int64_t)row * b.ldo - begin), r, b.f.inv_t, from, min(from + each, end), threadIdx.x, LP_THREADS);
            __syncthreads();
        });
    if (rows.offsets) asm volatile("griddepcontrol.wait;" ::: "memory");  // what comes next waits for both
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

// A row takes one CTA, or several where that is sooner: one of 128 threads takes 8 KB of a row in a microsecond, all of them together 6 GB in a millisecond, and joining the parts 15 us and
// 0.07 for each row (300 rows of 100,000 bfloat16 36 us in one CTA each and 49 in several; 600 of 1M 264 and 240).  total: entries of all lists; size: bytes of one.
inline LpPlan lp_plan(int m, int64_t cols, int64_t total, bool lists, int size, int sm_count) {
    LpPlan p;
    const int64_t entries = lists ? total : (int64_t)m * cols, mean = m ? entries / m : 0;
    p.split = mean > 16384 && (double)mean * size / 8200 > (double)entries * size / 6e6 + 15 + 0.07 * m;
    if (!p.split) return p;
    p.unit = 4096;
    while (p.unit < 32768 && entries / p.unit > 16ll * sm_count) p.unit *= 2;
    p.units_per_row = (int)(cols / p.unit + 2);
    p.units = lists ? (total + 16) / p.unit + m + 1 : (int64_t)m * p.units_per_row;
    p.chunks = lists ? (total + 16) / LP_LEAST_CHUNK + m + 1 : (int64_t)m * (cols / LP_LEAST_CHUNK + 2);
    return p;
}

// A launch behind a kernel that lets it begin at once (and was itself launched as usual, so that all that came before it is done): what the two do does not depend on the other but for
// what is behind a griddepcontrol.wait.
template <typename... P, typename... A>
inline void launch_beside(cudaStream_t stream, void (*kern)(P...), size_t grid, int threads, A... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CU_CHECK(launch_cast(cfg, kern, args...));
}

template <typename T>
inline void log_probs(const CtxPtr& c, const T* scores, LpArgs a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    a.rows.shift = (int64_t)((uintptr_t)scores / sizeof(T) % V);
    const T* x = scores - a.rows.shift;
    const LpPlan p = lp_plan(a.m, a.rows.cols, a.rows.total, a.rows.offsets != nullptr, sizeof(T), c->sm_count);
    if (!p.split) {
        // What follows the pass is mostly waits, which an SM hides among many rows.  With fewer rows than it takes, larger CTAs do (10,000 lists of 18,000 float32: 32 threads 211 us, 128
        // 239; 20,000 of 300: 72 and 170; 2,000 of 60,000: 307 and 137).  The bound of the k largest takes k threads.
        const int64_t mean = a.rows.offsets ? a.rows.total / a.m : a.rows.cols;
        int th = mean <= 1024 || (a.m >= 32 * c->sm_count && mean <= 32768) ? 32 : a.m >= 16 * c->sm_count && mean <= 16384 ? 64 : 128;
        while (th < a.k) th *= 2;
        auto kern = th == 32 ? log_probs_row_kernel<32, T> : th == 64 ? log_probs_row_kernel<64, T> : log_probs_row_kernel<128, T>;
        a.placed = a.ids && a.targets && (mean > 8192 || (a.rows.total > 1 << 18 && a.m <= 1 << 11));  // the second: lists that are long among others
        if (a.placed) {
            log_probs_places_kernel<<<(unsigned)std::min((a.m - 1) / LP_WARPS + 1, 8 * c->sm_count), LP_THREADS, 0, stream>>>(a);
            KERNEL_CHECK();
            launch_beside(stream, kern, (size_t)a.m, th, x, a);
            return;
        }
        kern<<<(unsigned)a.m, th, 0, stream>>>(x, a);
        KERNEL_CHECK();
        return;
    }
    if (workspace_bytes < p.bytes() || !workspace || ((uintptr_t)workspace & 15)) fail(CULSH_ERR_INVALID, "the workspace has to be %zu bytes, aligned to 16", p.bytes());
    if (p.units > 0x7FFFFFFFll) fail(CULSH_ERR_UNSUPPORTED, "%lld entries are too many for one call", (long long)a.rows.total);
    a.unit = p.unit;
    a.units_per_row = p.units_per_row;
    a.parts = static_cast<float4*>(workspace);
    a.maxima = reinterpret_cast<uint32_t*>(a.parts + p.units);
    launch_next(stream, log_probs_unit_kernel<T>, (size_t)p.units, (unsigned)LP_THREADS, 0, x, a);
    KERNEL_CHECK();
    launch_next(stream, log_probs_join_kernel<T>, (size_t)a.m, (unsigned)LP_THREADS, 0, x, a);
    KERNEL_CHECK();
}

template <typename T>
inline void log_probs_backward(const CtxPtr& c, const T* scores, T* out, LpBackward b, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    LpRows& r = b.f.rows;
    r.shift = (int64_t)((uintptr_t)scores / sizeof(T) % V);
    const int64_t mean = r.total / b.f.m;
    b.span = mean >= 1024 ? 512 : mean >= 64 ? 128 : 32;
    b.units = r.offsets ? (int64_t)ceil_div((size_t)(r.total + r.shift), (size_t)b.span) : r.cols / LP_ROW_SPAN<T> + 2;
    const size_t grid = r.offsets ? ceil_div((size_t)b.units, LP_WARPS) : (size_t)b.units * b.f.m;
    if (grid > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "too many entries for one call");
    const bool alike = (((uintptr_t)(out - r.shift) | (r.offsets ? 0u : (uintptr_t)((b.ldo - r.ld) * (int64_t)sizeof(T)))) & 15u) == 0;
    const T* const x = scores - r.shift;
    auto by = [&](auto form) {
        constexpr bool ALIKE = decltype(form)::value;
        if (r.offsets ? mean <= 512 && r.total <= LP_ALONE : r.cols <= LP_ALONE_ROW && b.f.m * r.cols <= LP_ALONE_ALL) {
            if (r.offsets) log_probs_backward_lists_kernel<ALIKE, true, T><<<(unsigned)grid, LP_THREADS, 0, stream>>>(x, out, b);
            else log_probs_backward_rows_kernel<ALIKE, true, T><<<(unsigned)grid, LP_THREADS, 0, stream>>>(x, out, b);
            KERNEL_CHECK();
            return;
        }
        b.whole = 4 * c->sm_count;
        b.shares = 1;
        while (b.shares < 16 && 2 * b.shares * ((b.f.m - 1) / LP_WARPS + 1) <= b.whole) b.shares *= 2;
        b.whole = std::min((b.f.m - 1) / LP_WARPS + 1, b.whole / b.shares) * b.shares;
        if (r.offsets) {
            log_probs_backward_lists_kernel<ALIKE, false, T><<<(unsigned)grid, LP_THREADS, 0, stream>>>(x, out, b);
            KERNEL_CHECK();
            launch_beside(stream, log_probs_backward_whole_kernel<ALIKE, T>, (size_t)b.whole, LP_THREADS, x, out, b);
        } else {
            log_probs_backward_whole_kernel<ALIKE, T><<<(unsigned)b.whole, LP_THREADS, 0, stream>>>(x, out, b);
            KERNEL_CHECK();
            launch_beside(stream, log_probs_backward_rows_kernel<ALIKE, false, T>, grid, LP_THREADS, x, out, b);
        }
    };
    if (alike) by(std::true_type());
    else by(std::false_type());
}

}  // namespace culsh_b200
