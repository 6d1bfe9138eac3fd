// Entry points of the ranking operators: rows in 4 bits, products and scores, log probabilities (see include/culsh_b200.h).
#include "entry.cuh"
#include "log_probs.cuh"
#include "mx_product.cuh"
#include "mx_rows.cuh"
#include "mx_score.cuh"

#include <algorithm>
#include <cmath>

using namespace culsh_b200;

namespace {

void check_rows(const void* codes, const void* scales, int n, int d) {
    need(n > 0 && d > 0, "rows and features must be positive");
    need(n <= 0x7FFFFF80, "at most 2,147,483,520 rows");
    need(d <= 1 << 20, "at most 1,048,576 features");
    need(codes && scales, "null argument");
    need((((uintptr_t)codes | (uintptr_t)scales) & 15) == 0, "codes and scales have to begin at a multiple of 16 bytes");
}
LpArgs log_probs_args(const void* scores, int m, int64_t cols, int64_t ld, const int64_t* offsets, const int32_t* ids, int64_t total, double temperature,
                      const int64_t* targets) {
    need(scores || (offsets && total == 0), "null argument");
    need(m > 0, "rows must be positive");
    need(temperature > 0 && std::isfinite(temperature), "temperature must be positive");
    need(temperature > 4.3e-39, "the temperature is too small: log2(e) by it has to be a float");
    if (offsets) {
        need(total >= 0, "total must not be negative");
        if (total >= (ids ? 1ll << 32 : 1ll << 31)) fail(CULSH_ERR_UNSUPPORTED, "%lld entries are too many for one call", (long long)total);  // places have 32 bits
        need(!(targets && !ids), "targets of lists need the lists' ids");
    } else {
        need(cols > 0 && cols < (1ll << 31), "columns must be positive and below 2^31");
        need(ld >= cols, "rows must not overlap");
        need(!ids, "ids belong to lists");
    }
    LpArgs a{};
    a.rows.offsets = offsets;
    a.rows.ld = ld;
    a.rows.cols = offsets ? 0 : cols;
    a.rows.total = offsets ? total : 0;
    a.ids = ids;
    a.targets = targets;
    a.m = m;
    a.c = (float)(1.4426950408889634 / temperature);
    a.inv_t = (float)(1 / temperature);
    return a;
}

}  // namespace

extern "C" {

int culsh_mx_quantize(culsh_handle* h, const void* X, int type, int n, int d, int64_t ld, uint8_t* codes, uint8_t* scales, float* norms, void* stream) {
    return guarded([&] {
        need(h && X && norms, "null argument");
        check_rows(codes, scales, n, d);
        need(ld >= d, "rows must not overlap");
        DeviceGuard g(h->ctx->device);
        by_type(type, ALL_TYPES, X, [&](auto* x) { mx_quantize(x, n, d, ld, codes, scales, norms, stream_of(stream)); });
    });
}

int culsh_mx_dequantize(culsh_handle* h, const uint8_t* codes, const uint8_t* scales, int n, int d, void* out, int type, void* stream) {
    return guarded([&] {
        need(h && out, "null argument");
        check_rows(codes, scales, n, d);
        DeviceGuard g(h->ctx->device);
        by_type(type, ALL_TYPES, out, [&](auto* o) { mx_dequantize(codes, scales, n, d, o, stream_of(stream)); });
    });
}

int culsh_mx_product(culsh_handle* h, const uint8_t* q_codes, const uint8_t* q_scales, const float* q_norms, int n_queries, const uint8_t* codes,
                     const uint8_t* scales, const float* norms, int n, int d, int metric, void* out, int type, int64_t ld, void* stream) {
    return guarded([&] {
        need(h && out && norms && q_norms, "null argument");
        check_rows(codes, scales, n, d);
        check_rows(q_codes, q_scales, n_queries, d);
        need(metric >= 0 && metric <= 2, "metric must be 0, 1 or 2");
        need(ld >= n, "rows must not overlap");
        DeviceGuard g(h->ctx->device);
        by_type(type, SCORE_TYPES, out, [&](auto* o) {
            if constexpr (!std::is_same<decltype(o), double*>::value)
                mx_product(h->ctx, q_codes, q_scales, q_norms, n_queries, codes, scales, norms, n, d, metric, o, ld, wait_word(h->ctx), stream_of(stream));
        });
    });
}

int culsh_mx_product_dense(culsh_handle* h, const void* Q, int q_type, int n_queries, int64_t ldq, const uint8_t* codes, const uint8_t* scales,
                           const float* norms, int n, int d, int metric, void* out, int type, int64_t ld, void* workspace, uint64_t workspace_bytes,
                           void* stream) {
    return guarded([&] {
        need(h && Q && out && norms, "null argument");
        check_rows(codes, scales, n, d);
        need(n_queries > 0, "queries must be positive");
        need(metric >= 0 && metric <= 2, "metric must be 0, 1 or 2");
        need(ld >= n && ldq >= d, "rows must not overlap");
        need_workspace(workspace, workspace_bytes, mx_bytes(n_queries, d));
        DeviceGuard g(h->ctx->device);
        uint8_t* const q_codes = static_cast<uint8_t*>(workspace);
        uint8_t* const q_scales = q_codes + (size_t)n_queries * mx_groups(d) * (MX_GROUP / 2);
        float* const q_norms = reinterpret_cast<float*>(q_scales + (size_t)mx_tiles(n_queries) * mx_groups(d) * MX_TILE_BYTES);
        by_type(type, SCORE_TYPES, out, [&](auto* o) {
            if constexpr (!std::is_same<decltype(o), double*>::value) {
                by_type(q_type, ALL_TYPES, Q, [&](auto* q) { mx_quantize(q, n_queries, d, ldq, q_codes, q_scales, q_norms, stream_of(stream)); });
                mx_product(h->ctx, q_codes, q_scales, q_norms, n_queries, codes, scales, norms, n, d, metric, o, ld, wait_word(h->ctx), stream_of(stream));
            }
        });
    });
}

int culsh_mx_product_check(culsh_handle* h, void* stream) {
    return guarded([&] {
        need(h, "null handle");
        DeviceGuard g(h->ctx->device);
        int word = 0;
        CU_CHECK(cudaMemcpyAsync(&word, wait_word(h->ctx), sizeof(word), cudaMemcpyDeviceToHost, stream_of(stream)));
        CU_CHECK(cudaStreamSynchronize(stream_of(stream)));
        if (!word) return;
        CU_CHECK(cudaMemsetAsync(wait_word(h->ctx), 0, sizeof(word), stream_of(stream)));
        fail(CULSH_ERR_INTERNAL, "a wait in a product or in scores ran out of time; what they should have made is NaN");
    });
}

int culsh_mx_score_workspace(culsh_handle* h, int n_queries, int d, int64_t total, uint64_t* bytes) {
    return guarded([&] {
        need(h && bytes, "null argument");
        need(n_queries >= 0 && d > 0 && total >= 0, "sizes must not be negative");
        *bytes = total ? mx_score_workspace(n_queries, d, total) : 0;
    });
}

int culsh_mx_score(culsh_handle* h, const void* Q, int type, int n_queries, int64_t ldq, const uint8_t* codes, const uint8_t* scales, const float* norms,
                   int n, int d, int metric, const int32_t* ids, const int64_t* offsets, int64_t total, float* out, void* workspace,
                   uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(h && Q && norms && offsets && (total == 0 || (ids && out)), "null argument");
        check_rows(codes, scales, n, d);
        need(n_queries > 0, "queries must be positive");
        need(metric >= 0 && metric <= 2, "metric must be 0, 1 or 2");
        need(ldq >= d, "rows must not overlap");
        need(total >= 0, "total must not be negative");
        if (total == 0) return;
        need_workspace(workspace, workspace_bytes, mx_score_workspace(n_queries, d, total));
        DeviceGuard g(h->ctx->device);
        MxScoreArgs a{};
        a.codes = codes, a.scales = scales, a.norms = norms, a.ids = ids, a.offsets = offsets, a.out = out;
        a.ldq = ldq, a.total = total, a.n = n, a.nq = n_queries, a.d = d, a.groups = mx_groups(d), a.metric = metric;
        by_type(type, ALL_TYPES, Q, [&](auto* q) { mx_score(h->ctx, q, a, workspace, wait_word(h->ctx), stream_of(stream)); });
    });
}

int culsh_candidates_after(culsh_handle* h, const culsh_candidates* c, void* stream) {
    return guarded([&] {
        need(h && c, "null argument");
        DeviceGuard g(c->ctx->device);
        cudaStreamCaptureStatus capture;
        CU_CHECK(cudaStreamIsCapturing(stream_of(stream), &capture));
        if (capture != cudaStreamCaptureStatusNone) return;  // a wait would make the engine's stream part of the graph
        std::lock_guard<std::mutex> lock(c->ctx->read_by_lock);
        CU_CHECK(cudaEventRecord(c->ctx->read_by, stream_of(stream)));
        CU_CHECK(cudaStreamWaitEvent(c->ctx->stream, c->ctx->read_by, 0));
    });
}

int culsh_log_probs_workspace(culsh_handle* h, int type, int m, int64_t cols, int is_lists, int64_t total, uint64_t* bytes) {
    return guarded([&] {
        need(h && bytes, "null argument");
        need(m > 0 && cols >= 0 && total >= 0, "sizes must not be negative");
        *bytes = lp_plan(m, cols, total, is_lists != 0, type == CULSH_F32 ? 4 : 2, h->ctx->sm_count).bytes();
    });
}

int culsh_log_probs(culsh_handle* h, const void* scores, int type, int m, int64_t cols, int64_t ld, const int64_t* offsets, const int32_t* ids,
                    int64_t total, double temperature, const int64_t* targets, int k, float* log_probs_out, float* entropy, float* lse,
                    float* top_log_probs, int32_t* top_ids, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(h && entropy && lse, "null argument");
        need(k >= 0 && k <= LP_MAX_K, "k must be between 0 and 128");
        need(k == 0 || (top_log_probs && top_ids), "null argument");
        need(!targets || log_probs_out, "null argument");
        LpArgs a = log_probs_args(scores, m, cols, ld, offsets, ids, total, temperature, targets);
        a.k = k, a.log_probs = log_probs_out, a.entropy = entropy, a.lse = lse, a.top_log_probs = top_log_probs, a.top_ids = top_ids;
        DeviceGuard g(h->ctx->device);
        by_type(type, SCORE_TYPES, scores, [&](auto* s) {
            if constexpr (!std::is_same<decltype(s), const double*>::value) log_probs(h->ctx, s, a, workspace, workspace_bytes, stream_of(stream));
        });
    });
}

int culsh_log_probs_backward(culsh_handle* h, const void* scores, int type, int m, int64_t cols, int64_t ld, const int64_t* offsets,
                             const int32_t* ids, int64_t total, double temperature, const int64_t* targets, const float* lse, const float* entropy,
                             const float* grad_log_probs, const float* grad_entropy, void* grad_scores, int64_t ld_grad, void* stream) {
    return guarded([&] {
        need(h && lse && entropy, "null argument");
        need(!grad_log_probs || targets, "the gradient of log probabilities needs their targets");
        LpBackward b{};
        b.f = log_probs_args(scores, m, cols, ld, offsets, ids, total, temperature, targets);
        if (offsets && total == 0) return;
        need(grad_scores, "null argument");
        need(offsets || ld_grad >= cols, "rows must not overlap");
        b.ldo = ld_grad;
        b.lse = lse, b.entropy = entropy, b.g = grad_log_probs, b.h = grad_entropy;
        DeviceGuard g(h->ctx->device);
        by_type(type, SCORE_TYPES, scores, [&](auto* s) {
            using T = std::remove_const_t<std::remove_pointer_t<decltype(s)>>;
            if constexpr (!std::is_same<T, double>::value) log_probs_backward(h->ctx, s, static_cast<T*>(grad_scores), b, stream_of(stream));
        });
    });
}

}  // extern "C"
