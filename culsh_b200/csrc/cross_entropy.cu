// Entry points of the softmax cross entropy over every row (see include/culsh_b200.h).
#include <cmath>

#include "cross_entropy.cuh"
#include "entry.cuh"

using namespace culsh_b200;

namespace {

CeCall call_of(culsh_handle* h, const void* Q, int64_t ldq, const void* X, int64_t ldx, int type, int m, int n, int d, const int64_t* targets, const float* bias,
               double temperature, void* stream) {
    need(h && Q && X, "null argument");
    need(type >= 0 && type <= 3 && (SCORE_TYPES >> type & 1), "queries and rows have to be float32, float16 or bfloat16");
    need(m > 0 && n > 0 && d > 0, "queries, rows and features must be positive");
    need(m <= 0x7FFF0000 && n <= 0x7FFF0000, "at most 2,147,418,112 queries and rows");  // places a tile behind the last one are still below 2^31
    need(d <= 1 << 16, "at most 65,536 features");
    need(ldq >= d && ldx >= d, "rows must not overlap");
    need(temperature > 0 && std::isfinite(temperature), "temperature must be positive");
    need(temperature > 4.3e-39, "the temperature is too small: log2(e) by it has to be a float");
    CeCall k{};
    k.c = h->ctx, k.Q = Q, k.X = X, k.ldq = ldq, k.ldx = ldx, k.type = type, k.m = m, k.n = n, k.d = d;
    k.targets = targets, k.bias = bias, k.temperature = temperature, k.d_error = wait_word(h->ctx), k.stream = stream_of(stream);
    return k;
}

}  // namespace

extern "C" {

int culsh_cross_entropy_workspace(culsh_handle* h, const void* Q, int64_t ldq, const void* X, int64_t ldx, int type, int m, int n, int d, int has_bias, int gradients,
                                  uint64_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        need(gradients >= 0 && gradients <= 3, "gradients must be between 0 and 3");
        static const float some = 0.f;
        const CeCall k = call_of(h, Q, ldq, X, ldx, type, m, n, d, nullptr, has_bias ? &some : nullptr, 1., nullptr);
        *bytes = CePlan(k, gradients != 0, gradients & 1, gradients & 2, nullptr).space.used;
    });
}

int culsh_cross_entropy(culsh_handle* h, const void* Q, int64_t ldq, const void* X, int64_t ldx, int type, int m, int n, int d, const int64_t* targets, const float* bias,
                        double temperature, float* losses, float* lse, float* lse_low, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const CeCall k = call_of(h, Q, ldq, X, ldx, type, m, n, d, targets, bias, temperature, stream);
        need(losses && lse && lse_low, "null argument");
        need_workspace(workspace, workspace_bytes, CePlan(k, false, false, false, nullptr).space.used);
        DeviceGuard g(h->ctx->device);
        cross_entropy(k, losses, lse, lse_low, workspace);
    });
}

int culsh_cross_entropy_backward(culsh_handle* h, const void* Q, int64_t ldq, const void* X, int64_t ldx, int type, int m, int n, int d, const int64_t* targets,
                                 const float* bias, double temperature, const float* losses, const float* lse, const float* lse_low, const float* grad_losses,
                                 const float* grad_lse, void* grad_Q, int64_t ld_gq, void* grad_X, int64_t ld_gx, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const CeCall k = call_of(h, Q, ldq, X, ldx, type, m, n, d, targets, bias, temperature, stream);
        need(losses && lse && lse_low, "null argument");
        need(!grad_losses || targets, "the gradient of losses needs their targets");
        need(!(grad_Q && ld_gq < d) && !(grad_X && ld_gx < d), "rows must not overlap");
        if (!grad_Q && !grad_X) return;
        need_workspace(workspace, workspace_bytes, CePlan(k, true, grad_Q != nullptr, grad_X != nullptr, nullptr).space.used);
        DeviceGuard g(h->ctx->device);
        by_type(type, SCORE_TYPES, Q, [&](auto* q) {
            using T = std::remove_const_t<std::remove_pointer_t<decltype(q)>>;
            if constexpr (!std::is_same<T, double>::value)
                cross_entropy_backward<T>(k, losses, lse, lse_low, grad_losses, grad_lse, static_cast<T*>(grad_Q), ld_gq, static_cast<T*>(grad_X), ld_gx, workspace);
        });
    });
}

}  // extern "C"
