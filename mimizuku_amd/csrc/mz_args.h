// What the C entry points check their arguments with.
#pragma once
#include <algorithm>

#include "../../include/mimizuku.h"
#include "mz_internal.h"

#define DP(T, x) ((T*)(uintptr_t)(x))

// The context's device is current while a call runs, whatever was before and will be after.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if ((status_ = mz_hip(hipGetDevice(&before_), "hipGetDevice"))) return;
        if (before_ == device) before_ = -1;
        else status_ = mz_hip(hipSetDevice(device), "hipSetDevice");
    }
    ~OnDevice() {
        if (before_ >= 0) hipSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    int status() const { return status_; }

private:
    int before_ = -1, status_ = MZ_OK;
};

inline bool aligned(uint64_t p, uint64_t n) { return p % n == 0; }

// Elements of each tensor stay below this, so that no 64-bit byte offset of a kernel can wrap.
constexpr int64_t MOST = (int64_t)1 << 46;

// Offsets of rows x tokens x heads 64-channel rows: in range, and multiples of 8 elements.
inline bool strides_ok(const int64_t (&stride)[3], const int64_t (&n)[3]) {
    for (int i = 0; i < 3; i++)
        if (stride[i] < 0 || stride[i] % 8 || stride[i] > MOST || (n[i] > 1 && stride[i] > MOST / (n[i] - 1))) return false;
    return true;
}

// Whether those rows lie apart from each other, each dimension's steps outside what the smaller ones span.
inline bool apart(const int64_t (&stride)[3], const int64_t (&n)[3]) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
    int64_t span = 64;
    for (int i : order) {
        if (n[i] <= 1) continue;
        if (stride[i] < span) return false;
        span += stride[i] * (n[i] - 1);
    }
    return true;
}

inline int check_work(const char* who, uint64_t work, size_t have, size_t need) {
    if (need && (!work || !aligned(work, 256) || have < need))
        return mz_fail(MZ_ERR_ARG, "%s: needs a workspace of %zu bytes, aligned to 256 (given %zu)", who, need, work ? have : (size_t)0);
    return MZ_OK;
}
