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
// The product with the reciprocal is up to 2^-16 off the quotient; where that leaves a choice, the quotient itself is rounded.
template <typename T>
__device__ __forceinline__ int i8_code(T x, float scale, float inv) {
    const float q = (float)x * inv, k = rintf(q);
    if (fabsf(fabsf(q - k) - 0.5f) < 6.103515625e-5f) return (int)rint((double)x / (double)scale);
    return (int)k;
}
template <>
__device__ __forceinline__ int i8_code<double>(double x, float scale, float) {
    return (int)rint(x / (double)scale);
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
// rows are read twice.  n d z read, n (d + 8) written.
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
#pragma unroll
        for (int i = 0; i < I8_VECS; ++i) {
            const int c = c0 + i * step + at * V;
            alignas(8) int8_t k[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int code = none ? 0 : i8_code<T>(held[i].v[j], scale, inv);
                k[j] = (int8_t)code;
                sum += code * code;
            }
            if (in && c < pitch) {  // a multiple of 16, as c is one of V
                if (V == 8) *reinterpret_cast<uint2*>(o + c) = *reinterpret_cast<const uint2*>(k);
                else *reinterpret_cast<uint32_t*>(o + c) = *reinterpret_cast<const uint32_t*>(k);
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

// Four codes to a thread.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) i8_dequantize_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int n, int d, T* __restrict__ out) {
    const int words = (d + 3) / 4;
    const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, row = unit / words;
    if (row >= n) return;
    const int c = (int)(unit - row * words) * 4;
    const char4 k = __ldg(reinterpret_cast<const char4*>(codes + row * (int64_t)i8_pitch(d) + c));
    using F = std::conditional_t<std::is_same<T, double>::value, double, float>;
    const F s = (F)__ldg(scales + row);
    struct alignas(4 * sizeof(T) > 16 ? 16 : 4 * sizeof(T)) Four { T v[4]; };
    const Four w = {{(T)((F)k.x * s), (T)((F)k.y * s), (T)((F)k.z * s), (T)((F)k.w * s)}};
    T* const o = out + row * (int64_t)d + c;
    if (VEC) {
        *reinterpret_cast<Four*>(o) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < d) o[i] = w.v[i];
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
    const size_t grid = ceil_div((size_t)n * ((d + 3) / 4), 256);
    if (grid > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "%d rows of %d values are too many", n, d);
    if (d % 4 == 0 && aligned16(out, 0)) i8_dequantize_kernel<T, true><<<(unsigned)grid, 256, 0, stream>>>(codes, scales, n, d, out);
    else i8_dequantize_kernel<T, false><<<(unsigned)grid, 256, 0, stream>>>(codes, scales, n, d, out);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
