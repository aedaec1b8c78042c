// What the entry points of the C ABI share: the calling thread's error message, launch checks and launch timing.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gdn {

// Sets the message of gdn_last_error() and returns code; clear_error empties it.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();

// After a launch: reports launch errors, and with GDN_DEBUG_SYNC=1 synchronises and reports execution errors.
int check_launch(hipStream_t st, const char *what);

// Brackets the launches of its scope with two events while gdn_profile_enable is on.
struct Timed {
    const char *name;
    hipStream_t st;
    hipEvent_t start = nullptr, stop = nullptr;
    Timed(const char *n, hipStream_t s);
    ~Timed();
    Timed(const Timed &) = delete;
    Timed &operator=(const Timed &) = delete;
};

// A launch has less than 2^32 threads along a dimension: a grid of `blocks` workgroups (less than 2^32), in rows if they are
// many.  The last row may be longer than what is left; block_index() of those is `blocks` or more.
inline dim3 grid_of(int64_t blocks) {
    constexpr int64_t ROW = 1 << 16;
    return blocks <= 1 << 21 ? dim3((unsigned)blocks) : dim3((unsigned)ROW, (unsigned)((blocks + ROW - 1) / ROW));
}
__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

inline size_t align_up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace gdn
