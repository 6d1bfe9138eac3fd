// What the entry points of the C ABI share: the objects behind its pointers, the errors that reach the caller as status codes, and
// the device that a call runs on.
#pragma once

#include "common.cuh"

// -----------------------------------------------------------------------------------------
// Objects behind the opaque pointers
// -----------------------------------------------------------------------------------------
struct culsh_handle {
    culsh_b200::CtxPtr ctx;
};

struct culsh_candidates {
    culsh_b200::CtxPtr ctx;
    int n_queries = 0;
    uint64_t total = 0;
    culsh_b200::DevBuf<int32_t> indices;
    culsh_b200::DevBuf<uint64_t> counts;
    culsh_b200::DevBuf<uint64_t> offsets;
    bool empty() const { return !indices.p && !counts.p && !offsets.p; }
};

namespace culsh_b200 {

inline thread_local std::string g_last_error;

template <typename F>
inline int guarded(F&& f) {
    try {
        f();
        return CULSH_OK;
    } catch (const Error& e) {
        g_last_error = e.what();
        return e.status;
    } catch (const std::bad_alloc&) {
        g_last_error = "host allocation failed";
        return CULSH_ERR_ALLOC;
    } catch (const std::exception& e) {
        g_last_error = e.what();
        return CULSH_ERR_INTERNAL;
    }
}

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        CU_CHECK(cudaGetDevice(&prev));
        if (prev != dev) CU_CHECK(cudaSetDevice(dev));
        else prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

}  // namespace culsh_b200
