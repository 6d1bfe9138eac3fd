// Rows in microscaled 4-bit floating point, and back.
//
// A row's values go in blocks of 32 that share a power of two: with a block's largest magnitude m,
//   E = clamp(floor(log2 m) - 2, -127, 127),   code = nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6} to x / 2^E (ties to the even code, beyond 6 to 6),
// and the value that is held is code * 2^E (the OCP microscaling formats' MXFP4: E2M1 elements, E8M0 scales).  m / 2^E lies in [4, 8).
// The division is exact, so the code is the one rounding.  A block with a NaN or an infinity gets the scale 255, which is NaN: such a row shows, it does not
// pass for another.
//
// Layout (mx_shape): codes row-major, two to a byte, the first in the low half, rows padded with zeros to groups of 128 values (64 bytes), which is what TMA
// loads and what a gathered row is read in.  Scales lie as the tensor cores take them: for 128 rows by 4 blocks (128 values) one tile of
// 512 bytes, byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4, so a row's four scales of a group are one aligned word and a tile goes into tensor memory as it is.
// norms[row] is the squared length of the row that is held, 0 for a row of zeros alone: MX_LEAST for what is too small for a square in 32 bits, infinite for what is too large.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace culsh_b200 {

constexpr float MX_LEAST = 1.401298464e-45f;  // 2^-149
constexpr int MX_BLOCK = 32, MX_GROUP = 128, MX_TILE_ROWS = 128, MX_TILE_BYTES = 512;

// Host and device: groups of 128 values in a row of d, tiles of 128 rows.
__host__ __device__ __forceinline__ int mx_groups(int d) { return (int)(((unsigned)d + (MX_GROUP - 1)) / MX_GROUP); }
__host__ __device__ __forceinline__ unsigned mx_tiles(int n) { return ((unsigned)n + (MX_TILE_ROWS - 1)) / MX_TILE_ROWS; }
// Offset in bytes of a row's scale word of a group.
__device__ __forceinline__ size_t mx_scale_at(int64_t row, int groups, int group) {
    return ((size_t)(row >> 7) * groups + group) * MX_TILE_BYTES + (size_t)((row & 31) * 16 + ((row >> 5) & 3) * 4);
}
// 2^(byte - 127); 0 is 2^-127, 255 NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7FFFFFFFu : byte == 0u ? 0x00400000u : byte << 23);
}
// The eight codes of a word as halves: codes 2i and 2i + 1 in h[i].  Exact.
__device__ __forceinline__ void mx_halves(uint32_t word, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
}
__device__ __forceinline__ float2 half_pair(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

__device__ __forceinline__ uint32_t mx_codes(const float (&y)[8]) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w;
}

// Eight values of a row from column c on, zeros behind its end.  VEC: 16-byte loads where all eight are there.  They go by L2, as everything does that a kernel that is
// launched early reads of what one in front may have written: a line of L1 can be from before its wait.
template <typename T, bool VEC>
struct EightOf {
    alignas(16) T v[8];
    __device__ __forceinline__ void load(const T* __restrict__ x, int c, int d) {
        if (VEC && c + 8 <= d) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<uint4*>(v)[i] = __ldcg(reinterpret_cast<const uint4*>(x + c) + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < d ? __ldcg(x + c + i) : T(0.f);
        }
    }
};

// Codes and scale of a block of 32 that four neighbouring lanes hold, eight values each.
template <typename T>
struct MxEncode {
    static __device__ __forceinline__ uint32_t codes(const T (&x)[8], uint32_t& scale) {
        float v[8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = (float)x[i];
            m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        }
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
        if (m >= 0x7F800000u) {
            scale = 255u;
            return 0u;
        }
        scale = (uint32_t)max((int)(m >> 23) - 2, 0);
        const float inv = __uint_as_float((254u - scale) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= inv;
        return mx_codes(v);
    }
};
template <>
struct MxEncode<double> {
    static __device__ __forceinline__ uint32_t codes(const double (&x)[8], uint32_t& scale) {
        unsigned long long m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, (unsigned long long)__double_as_longlong(x[i]) & 0x7FFFFFFFFFFFFFFFull);
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
        if (m >= 0x7FF0000000000000ull) {
            scale = 255u;
            return 0u;
        }
        scale = (uint32_t)min(max((int)(m >> 52) - 1023 - 2 + 127, 0), 254);
        const double inv = __longlong_as_double((long long)(1023 + 127 - (int)scale) << 52);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // cut to 24 bits, the last one set if anything was cut: the second rounding sees what side of a tie it is on
            const double y = x[i] * inv;
            v[i] = __double2float_rz(y);
            if ((double)v[i] != y) v[i] = __uint_as_float(__float_as_uint(v[i]) | 1u);
        }
        return mx_codes(v);
    }
};

// Sixteen lanes take a group of 128 values, eight each (four lanes a block); a row has `lanes` of them, 16 to 256, which step through its groups.
// n d z read, 17/32 n d + 4 n written (1M x 128 float32 130 us, 4.5 TB/s); bound by the issue of instructions (81 % of cycles, DRAM 48 %).  Rows behind the last one of the last tile get scales of 0.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const T* __restrict__ X, int n, int d, int64_t ld, int lanes, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, float* __restrict__ norms, KernelBefore before) {
    behind_kernel_before(X, codes, scales, norms, before);
    __shared__ float s_norm[8];
    const int groups = mx_groups(d), per_cta = 256 / lanes;
    const int64_t row = (int64_t)blockIdx.x * per_cta + threadIdx.x / lanes, rows = (int64_t)mx_tiles(n) * MX_TILE_ROWS;
    const int at = threadIdx.x % lanes;
    float norm = 0.f;
    for (int g0 = 0; g0 < groups; g0 += lanes / 16) {  // the same number of steps for all: lanes exchange values
        const int g = g0 + at / 16;
        EightOf<T, VEC> x;
        x.load(X + (row < n ? row : 0) * ld, row < n && g < groups ? g * MX_GROUP + (at & 15) * 8 : d, d);
        uint32_t scale;
        const uint32_t word = MxEncode<T>::codes(x.v, scale);
        uint32_t h[4];
        mx_halves(word, h);
        __half2 sum = __float2half2_rn(0.f);  // quarters up to 4 x 36: exact
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 c = *reinterpret_cast<const __half2*>(&h[i]);
            sum = __hfma2(c, c, sum);
        }
        const float2 s2 = __half22float2(sum);
        const float unit = mx_scale(scale);
        norm += (s2.x + s2.y) * unit * unit;
        // four blocks' scales in one word
        uint32_t four = scale << (8 * ((at >> 2) & 3));
        four |= __shfl_xor_sync(0xFFFFFFFFu, four, 4);
        four |= __shfl_xor_sync(0xFFFFFFFFu, four, 8);
        if (g < groups && row < rows) {
            if (row < n) *reinterpret_cast<uint32_t*>(codes + ((size_t)row * groups + g) * (MX_GROUP / 2) + (at & 15) * 4) = word;
            if ((at & 15) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_at(row, groups, g)) = row < n ? four : 0u;
        }
    }
    for (int o = 1; o < min(lanes, 32); o *= 2) norm += __shfl_xor_sync(0xFFFFFFFFu, norm, o);
    if (norm == 0.f) {  // for all lanes of the row in this warp: zeros, or too small for squares (from 2^-129 on the largest value is not rounded to 0)
        bool some = false;
        if (row < n)
            for (int g = at / 16; g < groups; g += lanes / 16)
                for (int c = g * MX_GROUP + (at & 15) * 8; c < min(g * MX_GROUP + (at & 15) * 8 + 8, d); ++c) some = some || fabsf((float)__ldcg(X + row * ld + c)) > 1.469367939e-39f;
        if (__any_sync(lanes == 16 ? 0xFFFFu << (threadIdx.x & 16) : 0xFFFFFFFFu, some)) norm = MX_LEAST;
    }
    if (lanes > 32) {
        if ((threadIdx.x & 31) == 0) s_norm[threadIdx.x >> 5] = norm;
        __syncthreads();
        if (at == 0) {
            norm = 0.f;
            for (int w = 0; w < lanes / 32; ++w) norm += s_norm[(threadIdx.x >> 5) + w];
        }
    }
    if (at == 0 && row < n) norms[row] = norm;
}

// Eight codes to a thread.  Bound by the stores' way out of the SMs (70 %, DRAM 40 %): 1M x 128 float32 123 us, written at 4.2 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int n, int d,
                                                            T* __restrict__ out) {
    const int groups = mx_groups(d);
    const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, row = unit / (groups * 16);
    if (row >= n) return;
    const int at = (int)(unit - row * (groups * 16)), c = at * 8;
    if (c >= d) return;
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(codes + (size_t)row * groups * (MX_GROUP / 2)) + at);
    const float s = mx_scale(__ldg(scales + mx_scale_at(row, groups, at >> 4) + ((at >> 2) & 3)));
    uint32_t h[4];
    mx_halves(word, h);
    using F = std::conditional_t<std::is_same<T, double>::value, double, float>;
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = half_pair(h[i]);
        v[2 * i] = (T)((F)f.x * (F)s);
        v[2 * i + 1] = (T)((F)f.y * (F)s);
    }
    T* o = out + (size_t)row * d + c;
    if (VEC && c + 8 <= d) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(o)[i] = reinterpret_cast<const uint4*>(v)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < d) o[i] = v[i];
    }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
// Bytes of n rows: codes, scales, norms, one behind the other.
inline size_t mx_bytes(int n, int d) { return (size_t)n * mx_groups(d) * (MX_GROUP / 2) + (size_t)mx_tiles(n) * mx_groups(d) * MX_TILE_BYTES + (size_t)n * 4; }

inline bool aligned16(const void* p, int64_t pitch_bytes) { return (((uintptr_t)p | (uintptr_t)pitch_bytes) & 15u) == 0; }

template <typename T>
inline void mx_quantize(const T* X, int n, int d, int64_t ld, uint8_t* codes, uint8_t* scales, float* norms, cudaStream_t stream) {
    int lanes = 16;
    while (lanes < 256 && lanes < 16 * mx_groups(d)) lanes *= 2;
    const unsigned grid = (unsigned)ceil_div((size_t)mx_tiles(n) * MX_TILE_ROWS, 256 / lanes);
    if (aligned16(X, ld * (int64_t)sizeof(T))) launch_next(stream, mx_quantize_kernel<T, true>, grid, 256u, 0, X, n, d, ld, lanes, codes, scales, norms);
    else launch_next(stream, mx_quantize_kernel<T, false>, grid, 256u, 0, X, n, d, ld, lanes, codes, scales, norms);
    KERNEL_CHECK();
}

template <typename T>
inline void mx_dequantize(const uint8_t* codes, const uint8_t* scales, int n, int d, T* out, cudaStream_t stream) {
    const size_t units = (size_t)n * mx_groups(d) * 16;
    auto kern = aligned16(out, d * (int64_t)sizeof(T)) ? mx_dequantize_kernel<T, true> : mx_dequantize_kernel<T, false>;
    if (ceil_div(units, 256) > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "%d rows of %d values are too many", n, d);
    kern<<<(unsigned)ceil_div(units, 256), 256, 0, stream>>>(codes, scales, n, d, out);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
