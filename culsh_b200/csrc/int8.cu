// Entry points of rows in 8-bit integers (see include/culsh_b200.h).
#include "entry.cuh"
#include "int8_product.cuh"

using namespace culsh_b200;

namespace {

void check_rows(const void* codes, const void* scales, const void* squares, int n, int d) {
    need(n > 0 && d > 0, "rows and features must be positive");
    need(n <= 0x7FFF0000, "at most 2,147,418,112 rows");  // places a tile behind the last one are still below 2^31
    need(d <= I8_MAX_FEATURES, "at most 131,072 features");
    need(codes && scales && squares, "null argument");
    need(((uintptr_t)codes & 15) == 0, "codes have to begin at a multiple of 16 bytes");
}
struct Held {
    int8_t* codes;
    float* scales;
    int32_t* squares;
    Held(void* workspace, int n, int d)
        : codes(static_cast<int8_t*>(workspace)), scales(reinterpret_cast<float*>(codes + (size_t)n * i8_pitch(d))), squares(reinterpret_cast<int32_t*>(scales + n)) {}
};

}  // namespace

extern "C" {

int culsh_i8_quantize(culsh_handle* h, const void* X, int type, int n, int d, int64_t ld, int8_t* codes, float* scales, int32_t* squares, void* stream) {
    return guarded([&] {
        need(h && X, "null argument");
        check_rows(codes, scales, squares, n, d);
        need(ld >= d, "rows must not overlap");
        DeviceGuard g(h->ctx->device);
        by_type(type, ALL_TYPES, X, [&](auto* x) { i8_quantize(x, n, d, ld, codes, scales, squares, stream_of(stream)); });
    });
}

int culsh_i8_dequantize(culsh_handle* h, const int8_t* codes, const float* scales, int n, int d, void* out, int type, void* stream) {
    return guarded([&] {
        need(h && out, "null argument");
        check_rows(codes, scales, scales, n, d);
        DeviceGuard g(h->ctx->device);
        by_type(type, ALL_TYPES, out, [&](auto* o) { i8_dequantize(codes, scales, n, d, o, stream_of(stream)); });
    });
}

int culsh_i8_product(culsh_handle* h, const int8_t* q_codes, const float* q_scales, const int32_t* q_squares, int n_queries, const int8_t* codes, const float* scales,
                     const int32_t* squares, int n, int d, int metric, void* out, int type, int64_t ld, void* stream) {
    return guarded([&] {
        need(h && out, "null argument");
        check_rows(codes, scales, squares, n, d);
        check_rows(q_codes, q_scales, q_squares, n_queries, d);
        need(metric >= 0 && metric <= 2, "metric must be 0, 1 or 2");
        need(ld >= n, "rows must not overlap");
        DeviceGuard g(h->ctx->device);
        by_type(type, SCORE_TYPES, out, [&](auto* o) {
            if constexpr (!std::is_same<decltype(o), double*>::value)
                i8_product(h->ctx, q_codes, q_scales, q_squares, n_queries, codes, scales, squares, n, d, metric, o, ld, wait_word(h->ctx), stream_of(stream));
        });
    });
}

int culsh_i8_product_dense(culsh_handle* h, const void* Q, int q_type, int n_queries, int64_t ldq, const int8_t* codes, const float* scales, const int32_t* squares, int n,
                           int d, int metric, void* out, int type, int64_t ld, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(h && Q && out, "null argument");
        check_rows(codes, scales, squares, n, d);
        need(n_queries > 0, "queries must be positive");
        need(metric >= 0 && metric <= 2, "metric must be 0, 1 or 2");
        need(ld >= n && ldq >= d, "rows must not overlap");
        need_workspace(workspace, workspace_bytes, i8_bytes(n_queries, d));
        DeviceGuard g(h->ctx->device);
        const Held q(workspace, n_queries, d);
        by_type(type, SCORE_TYPES, out, [&](auto* o) {
            if constexpr (!std::is_same<decltype(o), double*>::value) {
                by_type(q_type, ALL_TYPES, Q, [&](auto* x) { i8_quantize(x, n_queries, d, ldq, q.codes, q.scales, q.squares, stream_of(stream)); });
                i8_product(h->ctx, q.codes, q.scales, q.squares, n_queries, codes, scales, squares, n, d, metric, o, ld, wait_word(h->ctx), stream_of(stream));
            }
        });
    });
}

int culsh_i8_score(culsh_handle* h, const void* Q, int type, int n_queries, int64_t ldq, const int8_t* codes, const float* scales, const int32_t* squares, int n, int d,
                   int metric, const int32_t* ids, const int64_t* offsets, int64_t total, float* out, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        need(h && Q && offsets && (total == 0 || (ids && out)), "null argument");
        check_rows(codes, scales, squares, n, d);
        need(n_queries > 0, "queries must be positive");
        need(metric >= 0 && metric <= 2, "metric must be 0, 1 or 2");
        need(ldq >= d, "rows must not overlap");
        need(total >= 0, "total must not be negative");
        if (total == 0) return;
        need_workspace(workspace, workspace_bytes, i8_bytes(n_queries, d));
        DeviceGuard g(h->ctx->device);
        const Held q(workspace, n_queries, d);
        by_type(type, ALL_TYPES, Q, [&](auto* x) { i8_quantize(x, n_queries, d, ldq, q.codes, q.scales, q.squares, stream_of(stream)); });
        I8ScoreArgs a{};
        a.codes = codes, a.q_codes = q.codes, a.scales = scales, a.q_scales = q.scales, a.squares = squares, a.q_squares = q.squares;
        a.ids = ids, a.offsets = offsets, a.out = out, a.total = total, a.n = n, a.nq = n_queries, a.pitch = i8_pitch(d), a.metric = metric;
        i8_score_lists(h->ctx, a, stream_of(stream));
    });
}

}  // extern "C"
