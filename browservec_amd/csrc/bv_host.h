// What the host side's files share: the device handle, the error message of a
// failed call and growing device buffers.
#pragma once

#include "../../include/browservec_hip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>

struct bv_device {
    int ordinal = 0;
    hipDeviceProp_t prop{};
    bool lost = false;
    bool inject_append_oom = false;  // bv_debug_inject: fail the next append's allocation
    bool inject_append_late = false; // bv_debug_inject: fail the next append after its rows are encoded
    bool inject_slots_oom = false;   // bv_debug_inject: fail the next slot scan's allocation
    void *scratch = nullptr;         // this GPU's copy of the no-allocation scratch array
};

namespace bvk {
// Leaves the message for bv_last_error() and returns the code.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
// The same for a failed HIP call; errors that end the context mark the device lost.
int hip_fail(bv_device *dev, hipError_t e, const char *what);

#define HIPX(dev, expr, what)                        \
    do {                                             \
        hipError_t _e = (expr);                      \
        if (_e != hipSuccess) return hip_fail((dev), _e, (what)); \
    } while (0)

// -------------------------------------------------------- device buffers
struct DevBuf {
    void *p = nullptr;
    size_t cap = 0;
    ~DevBuf() { release(); }
    void release() {
        if (p) (void)hipFree(p);
        p = nullptr;
        cap = 0;
    }
    // Grow to at least `bytes`, preserving the first `keep` bytes.
    hipError_t ensure(size_t bytes, size_t keep, hipStream_t s, bool geometric = true) {
        if (bytes <= cap) return hipSuccess;
        size_t ncap = geometric ? std::max(bytes, cap + cap / 2) : bytes;
        ncap = (ncap + 255) & ~size_t(255);
        void *np = nullptr;
        hipError_t e = hipMalloc(&np, ncap);
        if (e != hipSuccess) return e;
        if (p && keep) {
            e = hipMemcpyAsync(np, p, keep, hipMemcpyDeviceToDevice, s);
            if (e == hipSuccess) e = hipStreamSynchronize(s);
            if (e != hipSuccess) {
                (void)hipFree(np);
                return e;
            }
        }
        if (p) (void)hipFree(p);
        p = np;
        cap = ncap;
        return hipSuccess;
    }
    template <class T> T *as() const { return (T *)p; }
};
}  // namespace bvk
