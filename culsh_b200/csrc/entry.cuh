// What the entry points that take device memory and a stream share: types of arrays, checks of arguments.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "api.cuh"

namespace culsh_b200 {

// Calls f(pointer of the type) for one of the types that are allowed (a mask of 1 << type).
template <typename P, typename F>
void by_type(int type, unsigned allowed, P* p, F&& f) {
    if (type < 0 || type > 3 || !(allowed >> type & 1)) fail(CULSH_ERR_INVALID, "type %d is not supported here", type);
    constexpr bool in = std::is_const<P>::value;
    auto as = [&](auto t) {
        using T = decltype(t);
        return static_cast<std::conditional_t<in, const T*, T*>>(p);
    };
    if (type == CULSH_F32) f(as(float()));
    else if (type == CULSH_F16) f(as(__half()));
    else if (type == CULSH_BF16) f(as(__nv_bfloat16()));
    else f(as(double()));
}
constexpr unsigned ALL_TYPES = 15, SCORE_TYPES = 1u << CULSH_F32 | 1u << CULSH_F16 | 1u << CULSH_BF16;

inline void need(bool ok, const char* what) {
    if (!ok) fail(CULSH_ERR_INVALID, "%s", what);
}
inline void need_workspace(const void* p, uint64_t have, size_t bytes) {
    if (bytes && (have < bytes || !p || ((uintptr_t)p & 15))) fail(CULSH_ERR_INVALID, "the workspace has to be %zu bytes, aligned to 16", bytes);
}
inline cudaStream_t stream_of(void* stream) { return static_cast<cudaStream_t>(stream); }
inline int* wait_word(const CtxPtr& c) { return c->d_error + 6; }

}  // namespace culsh_b200
