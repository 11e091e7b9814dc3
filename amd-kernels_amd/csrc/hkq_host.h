// hkq_host.h -- host-side helpers for the C-ABI entry points: argument checks
// that set a thread-local message and return hipErrorInvalidValue, and a
// launch-status check after each kernel launch.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "hkq.h"

namespace hkq {
void set_error(const char* fmt, ...);
int fail_arg(const char* file, int line, const char* msg);
int cu_count();

// An operand's memory: `rows` rows of `width` bytes, `pitch` bytes apart (p null: none).
struct MemRows {
    const void* p;
    int64_t rows, width, pitch;
};
// Whether two operands share a byte. Exact for one pitch (columns side by side
// in the rows of one buffer do not); rows of two pitches that lie in each other's
// range count as shared.
inline bool overlap(const MemRows& a, const MemRows& b) {
    if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
    const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p));
    auto extent = [](const MemRows& r) { return (__int128)(r.rows - 1) * r.pitch + r.width; };  // any pitch
    if (d >= extent(a) || -(__int128)d >= extent(b)) return false;
    const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    if (b.rows > 1 && b.pitch != pitch) return true;
    if (a.rows == 1 && b.rows == 1) return true;
    const int64_t col = (d % pitch + pitch) % pitch;  // b's first byte in a's rows
    return col < a.width || col + b.width > pitch;
}

// The dynamic LDS that a kernel takes, set once on each device (bit of `done`; a device
// past 63 every time).
template <class Kern>
inline int set_device_lds(Kern kern, int lds, std::atomic<uint64_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (e == hipSuccess && (done.load(std::memory_order_relaxed) & bit)) return 0;
    if (e == hipSuccess) e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
        set_error("hipFuncSetAttribute(MaxDynamicSharedMemorySize=%d) failed: %s", lds, hipGetErrorString(e));
        return (int)e;
    }
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}
}  // namespace hkq

#define HKQ_CHECK_ARG(cond, msg)                                     \
    do {                                                             \
        if (!(cond)) return ::hkq::fail_arg(__FILE__, __LINE__, msg); \
    } while (0)

#define HKQ_CHECK_ALIGN(ptr, a) \
    HKQ_CHECK_ARG((reinterpret_cast<uintptr_t>(ptr) % (a)) == 0, #ptr " must be " #a "-byte aligned")

// hipGetLastError after a launch: a bad configuration (grid too large, too much
// LDS) is reported here instead of silently dropping the work.
static inline int hkq_launch_status() {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) ::hkq::set_error("kernel launch failed: %s", hipGetErrorString(e));
    return (int)e;
}
