// What the host sources of libdeep_ep_hip.so share: errors in the reference's wording, the guard around every C entry, checks of
// tensor descriptors.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <exception>
#include <string>

#include "../../include/deep_ep_hip.h"

#define EP_INTERNAL __attribute__((visibility("hidden")))

// the thread's message for ep_last_error (ep_runtime.cpp)
EP_INTERNAL void ep_set_last_error(const char* message);
// <dir>/<name> of this library's code objects; dir == nullptr: the directory that holds the library
EP_INTERNAL std::string ep_code_object_path(const char* dir, const char* name);
// loads the kernels of ep_experts.hip (ep_experts.cpp); ep_init calls it
EP_INTERNAL void ep_load_expert_kernels(const char* dir);

namespace {

struct EpError {
    std::string msg;
};

inline std::string format(const char* fmt, ...) {
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return buf;
}

#define EP_HOST_ASSERT(cond)                                                                        \
    do {                                                                                            \
        if (!(cond)) throw EpError{format("Assertion exception (%s:%d): %s", __FILE_NAME__, __LINE__, #cond)}; \
    } while (0)

#define EP_HOST_UNREACHABLE(reason) \
    throw EpError { format("Assertion exception (%s:%d): %s", __FILE_NAME__, __LINE__, reason) }

#define HIP_CHECK(cmd)                                                                              \
    do {                                                                                            \
        const hipError_t e_ = (cmd);                                                                \
        if (e_ != hipSuccess)                                                                       \
            throw EpError{format("HIP runtime exception (%s:%d): Error code: %d, detail: %s", __FILE_NAME__, \
                                 __LINE__, (int)e_, hipGetErrorString(e_))};                        \
    } while (0)

template <class F>
int guarded(F&& f) {
    try {
        f();
        return 0;
    } catch (const EpError& e) {
        ep_set_last_error(e.msg.c_str());
        return 1;
    } catch (const std::exception& e) {
        ep_set_last_error(e.what());
        return 1;
    }
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// ---- tensor contracts -------------------------------------------------------------------------
inline bool present(const ep_tensor_t& t) { return t.data != nullptr; }

inline int elem_size(int dtype) {
    switch (dtype) {
        case EP_DTYPE_BF16: case EP_DTYPE_I16: return 2;
        case EP_DTYPE_FP8_E4M3: case EP_DTYPE_U8: return 1;
        case EP_DTYPE_I32: case EP_DTYPE_F32: return 4;
        case EP_DTYPE_I64: return 8;
        default: return 0;
    }
}

inline bool contiguous(const ep_tensor_t& t) {
    int64_t expect = 1;
    for (int d = t.ndim - 1; d >= 0; --d) {
        if (t.size[d] != 1 && t.stride[d] != expect) return false;
        expect *= t.size[d];
    }
    return true;
}

}  // namespace
