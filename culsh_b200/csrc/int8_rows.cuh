// Rows in 8-bit integers with a scale for each, and back.
//
//   scale = max(max |x| / 127 in 32 bits, 2^-126),   code = nearest whole number to x / scale, ties to the even one (-127 .. 127),
// and the value that is held is code * scale.  squares is the sum of a row's squared codes, exact in 32 bits (at most 131,072 values): cosines need no scale.  A row with a NaN or
// an infinity, or whose scale is beyond 32 bits, has the scale NaN, codes of 0 and squares of -1: it shows, it does not pass for another.
//
// Codes are row-major, rows padded with zeros to a multiple of 16, which is what TMA loads and what a gathered row is read in.
#pragma once

#include "mx_rows.cuh"

namespace culsh_b200 {

constexpr int I8_MAX_FEATURES = 1 << 17;
constexpr float I8_LEAST_SCALE = 1.175494351e-38f;  // 2^-126

__host__ __device__ __forceinline__ int i8_pitch(int d) { return (d + 15) & ~15; }

template <typename T>
struct I8Magnitude {  // as bits, which are in the values' order; NaNs above all
    using Bits = uint32_t;
    static constexpr Bits INF = 0x7F800000u;
    static __device__ __forceinline__ Bits of(T x) { return __float_as_uint((float)x) & 0x7FFFFFFFu; }
    static __device__ __forceinline__ float scale(Bits m) { return __fdiv_rn(__uint_as_float(m), 127.f); }
};
template <>
struct I8Magnitude<double> {
    using Bits = unsigned long long;
    static constexpr Bits INF = 0x7FF0000000000000ull;
    static __device__ __forceinline__ Bits of(double x) { return (Bits)__double_as_longlong(x) & 0x7FFFFFFFFFFFFFFFull; }
    static __device__ __forceinline__ float scale(Bits m) { return (float)(__longlong_as_double((long long)m) / 127.); }
};
// Four codes in a word.  A product with the reciprocal is up to 127 x 2^-23 (1.52e-5) off the quotient; the addition of 1.5 x 2^23 rounds it to a whole number, which is in the low bits.
// `far` is the largest distance from one: where it is so near a half that the quotient may lie on the other side, the caller has to look at what is left.
constexpr float I8_NEAR_HALF = 0.5f - 1.6e-5f;
__device__ __forceinline__ uint32_t i8_word(const uint32_t (&k)[4]) { return __byte_perm(__byte_perm(k[0], k[1], 0x0040), __byte_perm(k[2], k[3], 0x0040), 0x5410); }
template <typename T>
__device__ __forceinline__ uint32_t i8_codes(const T* x, float inv, float& far) {
    uint32_t k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = (float)x[i] * inv, t = q + 12582912.f;
        far = fmaxf(far, fabsf(q - (t - 12582912.f)));
        k[i] = __float_as_uint(t);
    }
    return i8_word(k);
}
// The same with each code the nearest: what x leaves over k * scale is, near half a scale, a multiple of 2^-24 of the scale's power of two, and so the fused multiply-add has no rounding;
// beyond a half the next number is nearer, at a half it is taken if it is the even one.
template <typename T>
__device__ __forceinline__ uint32_t i8_codes_near(const T* x, float scale, float inv) {
    uint32_t k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = (float)x[i], t = fmaf(v, inv, 12582912.f), left = fmaf(12582912.f - t, scale, v), half = 0.5f * scale;
        k[i] = __float_as_uint(t);
        if (fabsf(left) > half || (fabsf(left) == half && (k[i] & 1u))) k[i] += left > 0.f ? 1u : ~0u;
    }
    return i8_word(k);
}
template <>
__device__ __forceinline__ uint32_t i8_codes_near<double>(const double* x, float scale, float) {
    const double s = (double)scale;
    const uint32_t k[4] = {(uint32_t)(int)rint(x[0] / s), (uint32_t)(int)rint(x[1] / s), (uint32_t)(int)rint(x[2] / s), (uint32_t)(int)rint(x[3] / s)};
    return i8_word(k);
}

// V neighbouring values of a row, zeros behind its end.
template <typename T, int V, bool VEC>
struct SomeOf {
    alignas(16) T v[V];
    __device__ __forceinline__ void load(const T* __restrict__ x, int c, int d) {
        if (VEC && c + V <= d) {
#pragma unroll
            for (int i = 0; i < V * (int)sizeof(T) / 16; ++i) reinterpret_cast<uint4*>(v)[i] = __ldcg(reinterpret_cast<const uint4*>(x + c) + i);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = c + i < d ? __ldcg(x + c + i) : T(0.f);
        }
    }
};

// `lanes` threads (a power of two, 2 to 256) take a row, V values each of up to I8_VECS pieces of lanes * V, which stay in registers between the search for the largest and the codes; longer
// rows are read twice.  n d z read, n (d + 8) written; 1M x 128 float32 138 us, bound by issue (72 %) and HBM (57).  (Conversions and a look at each quotient 184.)
constexpr int I8_VECS = 4;
template <typename T>
struct I8Values { static constexpr int V = sizeof(T) == 2 ? 8 : 4; };

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) i8_quantize_kernel(const T* __restrict__ X, int n, int d, int64_t ld, int lanes, int8_t* __restrict__ codes, float* __restrict__ scales,
                                                          int32_t* __restrict__ squares, KernelBefore before) {
    behind_kernel_before(X, codes, scales, squares, before);
    using M = I8Magnitude<T>;
    using Bits = typename M::Bits;
    constexpr int V = I8Values<T>::V;
    __shared__ Bits s_top[8];
    __shared__ int s_sum[8];
    const int per_cta = 256 / lanes, at = threadIdx.x % lanes, pitch = i8_pitch(d), step = lanes * V;
    const int64_t row = (int64_t)blockIdx.x * per_cta + threadIdx.x / lanes;
    const bool in = row < n;
    const T* const x = X + (in ? row : 0) * ld;
    const int end = in ? d : 0;
    const bool once = d <= step * I8_VECS;
    SomeOf<T, V, VEC> held[I8_VECS];
    Bits top = 0;
    for (int c0 = 0; c0 < d; c0 += step * I8_VECS) {
#pragma unroll
        for (int i = 0; i < I8_VECS; ++i) held[i].load(x, c0 + i * step + at * V, end);
#pragma unroll
        for (int i = 0; i < I8_VECS; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) top = max(top, M::of(held[i].v[j]));
    }
    for (int o = 1; o < min(lanes, 32); o *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (lanes > 32) {
        if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
        __syncthreads();
        for (int w = 0; w < lanes / 32; ++w) top = max(top, s_top[(threadIdx.x / lanes) * (lanes / 32) + w]);
    }
    float scale = fmaxf(M::scale(top), I8_LEAST_SCALE);
    const bool none = top >= M::INF || !(scale < INFINITY);
    const float inv = none ? 0.f : 1.f / scale;
    int sum = 0;
    int8_t* const o = codes + (in ? row : 0) * (int64_t)pitch;
    for (int c0 = 0; c0 < pitch; c0 += step * I8_VECS) {
        if (!once) {
#pragma unroll
            for (int i = 0; i < I8_VECS; ++i) held[i].load(x, c0 + i * step + at * V, end);
        }
        uint32_t k[I8_VECS][V / 4];
        float far = 0.f;
#pragma unroll
        for (int i = 0; i < I8_VECS; ++i)
#pragma unroll
            for (int j = 0; j < V; j += 4) k[i][j / 4] = i8_codes(held[i].v + j, inv, far);
        if (std::is_same<T, double>::value || !(far < I8_NEAR_HALF)) {
#pragma unroll
            for (int i = 0; i < I8_VECS; ++i)
#pragma unroll
                for (int j = 0; j < V; j += 4) k[i][j / 4] = i8_codes_near(held[i].v + j, scale, inv);
        }
#pragma unroll
        for (int i = 0; i < I8_VECS; ++i) {
            const int c = c0 + i * step + at * V;
#pragma unroll
            for (int j = 0; j < V / 4; ++j) {
                if (none) k[i][j] = 0u;
                sum = __dp4a((int)k[i][j], (int)k[i][j], sum);
            }
            if (in && c < pitch) {  // a multiple of 16, as c is one of V
                if constexpr (V == 8) *reinterpret_cast<uint2*>(o + c) = make_uint2(k[i][0], k[i][1]);
                else *reinterpret_cast<uint32_t*>(o + c) = k[i][0];
            }
        }
    }
    for (int w = 1; w < min(lanes, 32); w *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, w);
    if (lanes > 32) {
        if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < lanes / 32; ++w) sum += s_sum[(threadIdx.x / lanes) * (lanes / 32) + w];
    }
    if (at == 0 && in) {
        scales[row] = none ? __int_as_float(0x7FFFFFFF) : scale;
        squares[row] = none ? -1 : sum;
    }
}

// Four times four codes to a thread.  A byte becomes a float as the low bits of one of 2^23 and more: conversions run at an eighth of the rate of additions.
// 1M x 128 float32 99 us, bound by HBM, which a fill of as many bytes keeps busy for 71.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) i8_dequantize_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t n, int d, T* __restrict__ out) {
    constexpr int EACH = 4;
    const unsigned words = (unsigned)(d + 3) / 4;
    const int64_t row0 = (int64_t)blockIdx.x * (256 * EACH) / words;
    const unsigned before = (unsigned)((int64_t)blockIdx.x * (256 * EACH) - row0 * words);
    using F = std::conditional_t<std::is_same<T, double>::value, double, float>;
    uint32_t k[EACH];
    F s[EACH];
    int64_t row[EACH];
    int c[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const unsigned at = before + threadIdx.x + i * 256, r = at / words;  // before < words <= 32,768
        row[i] = row0 + r;
        c[i] = (int)(at - r * words) * 4;
        k[i] = 0u, s[i] = 0;
        if (row[i] < n) {
            k[i] = __ldg(reinterpret_cast<const uint32_t*>(codes + row[i] * i8_pitch(d) + c[i]));
            s[i] = (F)__ldg(scales + row[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (row[i] >= n) continue;
        const uint32_t u = k[i] ^ 0x80808080u;
        struct alignas(4 * sizeof(T) > 16 ? 16 : 4 * sizeof(T)) Four { T v[4]; } w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w.v[j] = (T)((F)(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + j)) - 8388736.f) * s[i]);
        T* const o = out + row[i] * (int64_t)d + c[i];
        if (VEC) {
            *reinterpret_cast<Four*>(o) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c[i] + j < d) o[j] = w.v[j];
        }
    }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
// Bytes of n rows: codes, scales, squares, one behind the other.
inline size_t i8_bytes(int n, int d) { return (size_t)n * (i8_pitch(d) + 8); }

template <typename T>
inline void i8_quantize(const T* X, int n, int d, int64_t ld, int8_t* codes, float* scales, int32_t* squares, cudaStream_t stream) {
    constexpr int V = I8Values<T>::V;
    int lanes = 2;
    while (lanes < 256 && lanes * V * I8_VECS < d) lanes *= 2;
    const unsigned grid = (unsigned)ceil_div(n, 256 / lanes);
    if (aligned16(X, ld * (int64_t)sizeof(T))) launch_next(stream, i8_quantize_kernel<T, true>, grid, 256u, 0, X, n, d, ld, lanes, codes, scales, squares);
    else launch_next(stream, i8_quantize_kernel<T, false>, grid, 256u, 0, X, n, d, ld, lanes, codes, scales, squares);
    KERNEL_CHECK();
}

template <typename T>
inline void i8_dequantize(const int8_t* codes, const float* scales, int n, int d, T* out, cudaStream_t stream) {
    const size_t grid = ceil_div((size_t)n * ((d + 3) / 4), 1024);
    if (grid > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "%d rows of %d values are too many", n, d);
    if (d % 4 == 0 && aligned16(out, 0)) i8_dequantize_kernel<T, true><<<(unsigned)grid, 256, 0, stream>>>(codes, scales, n, d, out);
    else i8_dequantize_kernel<T, false><<<(unsigned)grid, 256, 0, stream>>>(codes, scales, n, d, out);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
