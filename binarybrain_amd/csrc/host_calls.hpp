// What the host sides of the entries share between their translation units: the last error, hints, the kernel timer, launches and workspaces.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <tuple>
#include <type_traits>

#pragma GCC visibility push(hidden)

namespace bbhip {

// the message of bbhip_GetLastErrorString; returns 1
int fail(char const *fmt, ...);

#define BBHIP_TRY(expr)                                                                              \
    do {                                                                                             \
        hipError_t e_ = (expr);                                                                      \
        if (e_ != hipSuccess) { return fail("%s: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); } \
    } while (0)

#define BBHIP_LAUNCH_CHECK() BBHIP_TRY(hipGetLastError())

// hints are for the next LUT call only: every entry spends them
void clear_hints(void);

// optional kernel timer: HIP events around the dominant kernel of each entry point, on the launch stream
enum TimedKernel : int { kTimeForward = 0, kTimeBackward = 1, kTimeBinary = 2, kTimeDx = 3, kTimeOther = 4, kTimedKinds = 5 };
struct TimedLaunch { hipEvent_t start, stop; int which; };
struct ScopedTimer {
    hipStream_t st; bool on; TimedLaunch t;
    ScopedTimer(int which, hipStream_t s, bool allowed = true);
    ~ScopedTimer();
};

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

inline bool starts_on_16_bytes(void const *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// an entry's workspace, as its ...WorkspaceBytes counts it
inline int check_workspace(void const *workspace, size_t size, size_t needed, char const *name)
{
    if (size < needed || (needed > 0 && workspace == nullptr)) { return fail("%s: a workspace of %zu bytes is needed, %zu given", name, needed, workspace ? size : (size_t)0); }
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)  { return fail("%s: the workspace must be aligned to 256 bytes", name); }
    return 0;
}

// A launch without the call-configuration stack and the copies that the <<<>>> form's host stub goes through: 2.7 us of host time for a kernel
// with 400 bytes of arguments instead of 3.2, and the host is what a program of small layers waits for.  Errors are read by BBHIP_LAUNCH_CHECK.
template <class... P, class... A>
void launch(void (*kernel)(P...), dim3 grid, dim3 block, unsigned lds_bytes, hipStream_t st, A const &... args)
{
    // an argument of the parameter's own type is passed where it lies
    std::tuple<std::conditional_t<std::is_same_v<P, A>, A const &, P>...> const held{args...};
    std::apply([&](auto const &... v) {
        void *where[] = {const_cast<void *>(static_cast<void const *>(&v))...};
        (void)hipLaunchKernel(reinterpret_cast<void const *>(kernel), grid, block, where, lds_bytes, st);
    }, held);
}

}  // namespace bbhip

#pragma GCC visibility pop
