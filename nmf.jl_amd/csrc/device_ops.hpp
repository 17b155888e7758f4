// device_ops.hpp -- what the entry points on device matrices (nmfx_xent*, nmfx_grad_norm, nmfx_clip_grad_norm) share: argument checks that
// turn into status codes, the thread's last message, the device switch, the launch check.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <exception>
#include <string>

#include "../../include/nmfx.h"

namespace nmfx {
namespace ops {

struct OpError {
    int status;
    std::string msg;
};
inline void require(bool ok, int status, const char *msg) {
    if (!ok) throw OpError{status, msg};
}
inline void hip_ok(hipError_t e, const char *what) {
    if (e != hipSuccess) throw OpError{NMFX_ERR_HIP, std::string("HIP error: ") + hipGetErrorString(e) + " at " + what};
}

// the calling thread's message (one per thread: operators have no context to keep it in)
std::string &last_error();

// the device of the operands, for the duration of a call
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        int n = 0;
        if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
            (void)hipGetLastError();
            throw OpError{NMFX_ERR_NO_DEVICE, "no HIP device visible: libnmfx has no CPU fallback"};
        }
        require(device >= 0 && device < n, NMFX_ERR_BAD_ARG, "device ordinal out of range");
        (void)hipGetLastError();      // an error that somebody else's call left behind is not a launch's of this one
        hip_ok(hipGetDevice(&before), "hipGetDevice");
        if (before != device) hip_ok(hipSetDevice(device), "hipSetDevice");
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

template <typename F> int guarded(F &&f) noexcept {
    try {
        f();
        last_error().clear();
        return NMFX_OK;
    } catch (const OpError &e) {
        try { last_error() = e.msg; } catch (...) {}
        return e.status;
    } catch (const std::exception &e) {
        try { last_error() = e.what(); } catch (...) {}
        return NMFX_ERR_STATE;
    } catch (...) {
        return NMFX_ERR_STATE;
    }
}

inline int elem_bytes(int dtype) {
    switch (dtype) {
        case NMFX_F32: return 4;
        case NMFX_F64: return 8;
        case NMFX_BF16: case NMFX_F16: return 2;
        default: return 0;
    }
}

struct View {           // a matrix as rows of contiguous elements
    char *p;
    int64_t rows, len, ld;   // len: elements of a row, ld: elements between rows
    int es, dtype;
    int64_t bytes() const { return ((rows - 1) * ld + len) * es; }
};

// whether two views have an element in common: exact where one is dense or both have one row stride, else "yes" where their extents overlap
inline bool meet(const View &a, const View &b) {
    if (!a.rows || !b.rows) return false;
    if (a.p > b.p) return meet(b, a);
    if (a.p + a.bytes() <= b.p) return false;
    const int64_t la = a.rows > 1 ? a.ld * a.es : 0, lb = b.rows > 1 ? b.ld * b.es : 0;
    if (!la || (lb && la != lb)) return true;
    const int64_t d = (b.p - a.p) % la;
    return !(d >= a.len * a.es && d + b.len * b.es <= la);
}

}  // namespace ops
}  // namespace nmfx
