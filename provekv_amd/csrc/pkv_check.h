// pkv_check.h -- what the host halves of the live-cache calls (pkv_attend.cpp,
// pkv_paged.cpp) check their arguments with, and the device they launch on.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>

#include "pkv_internal.h"

namespace pkv {
namespace {

using U128 = unsigned __int128;

inline int hip_rc(int e) {
    if (e == hipSuccess) return PKV_OK;
    return e == hipErrorOutOfMemory ? PKV_ERR_OOM : PKV_ERR_DEVICE;
}

// The context's device for the length of a call; the caller's current device
// comes back afterwards.
struct OnDevice {
    int was = -1, rc = PKV_OK;
    explicit OnDevice(int device) {
        if (hipGetDevice(&was) != hipSuccess) { rc = PKV_ERR_DEVICE; was = -1; return; }
        if (was == device) { was = -1; return; }
        if (hipSetDevice(device) != hipSuccess) rc = PKV_ERR_DEVICE;
    }
    ~OnDevice() {
        if (was >= 0) (void)hipSetDevice(was);
    }
};

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline uint64_t elem_bytes(int dtype) { return dtype == PKV_F32 ? 4 : 2; }

struct Axis {
    uint64_t stride;
    uint32_t count;
};
// Elements from the first row's start to the last row's end; 0: past 2^62.
inline uint64_t extent(const Axis* a, int n, uint64_t inner) {
    U128 e = inner;
    for (int i = 0; i < n; ++i) e += static_cast<U128>(a[i].stride) * (a[i].count - 1);
    return e >> 62 ? 0 : static_cast<uint64_t>(e);
}
// No two rows of `inner` elements share one: along every axis, in the order of
// their strides, a step is at least what the axes inside it span.
inline bool distinct(const Axis* a, int n, uint64_t inner) {
    Axis s[4];
    int m = 0;
    for (int i = 0; i < n; ++i)
        if (a[i].count > 1) s[m++] = a[i];
    std::sort(s, s + m, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
    U128 span = inner;
    for (int i = 0; i < m; ++i) {
        if (s[i].stride < span) return false;
        span += static_cast<U128>(s[i].stride) * (s[i].count - 1);
    }
    return true;
}
inline bool overlap(const void* a, uint64_t an, const void* b, uint64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}

constexpr uint32_t kMaxCount = 0x7fffffffu;
constexpr uint32_t kMaxRows = 1u << 30;   // query rows of all copies and query heads
// Elements from a slot to the next: a kernel's tile of 64 slots stays within
// 32-bit offsets of its first.
constexpr uint64_t kMaxSlotStride = 1u << 22;

}  // namespace
}  // namespace pkv
