// Scores of candidate lists: for every (query, candidate) pair of a CSR result the product of the query as it is with the row in microscaled 4-bit floating
// point (mx_rows.cuh), or the cosine, or the negative squared distance.  out[c] = sum_k q_k x^[id(c)]_k.
#pragma once

#include "mx_product.cuh"

namespace culsh_b200 {

// Largest i with offsets[i] <= at, i < n.
__device__ __forceinline__ int owner_of(const int64_t* __restrict__ offsets, int n, int64_t at) {
    int lo = 0, hi = n;  // offsets[lo] <= at < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(offsets + mid) <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

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

constexpr int MXS_PER_WARP = 64;

// A warp takes 64 neighbouring candidates, eight at a time; four lanes share one and take its blocks of 32 values (16 bytes) in turn.
template <typename T>
__global__ void __launch_bounds__(256) mx_score_kernel(const T* __restrict__ Q, MxScoreArgs a) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    int64_t at = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * MXS_PER_WARP;
    const int64_t end = min(at + MXS_PER_WARP, a.total);
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
            for (int i = lane; i < a.d; i += 32) {
                const float v = (float)x[i];
                q2 = fmaf(v, v, q2);
            }
            for (int o = 16; o; o >>= 1) q2 += __shfl_xor_sync(0xFFFFFFFFu, q2, o);
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
                else if (a.metric == MX_EUCLIDEAN) v = 2.f * dot - q2 - __ldg(a.norms + id);
                a.out[c] = v;
            }
        }
        at = last;
    }
}

template <typename T>
inline void mx_score(const T* Q, const MxScoreArgs& a, cudaStream_t stream) {
    const size_t grid = ceil_div((size_t)a.total, 8 * MXS_PER_WARP);
    if (grid > 0x7FFFFFFFull) fail(CULSH_ERR_UNSUPPORTED, "%lld candidates are too many for one call", (long long)a.total);
    mx_score_kernel<T><<<(unsigned)grid, 256, 0, stream>>>(Q, a);
    KERNEL_CHECK();
}

}  // namespace culsh_b200
