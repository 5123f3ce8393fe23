// Host checks and device element helpers shared by the described operators (op_rope.hip,
// op_linear.hip, op_cross_attention.hip).
#pragma once

#include <algorithm>
#include <cstdint>

#include "host.hpp"

namespace irodori {

inline size_t dtype_bytes(int dtype) { return dtype == IRODORI_DTYPE_F32 ? 4 : 2; }
inline bool op_dtype_ok(int dtype) {
    return dtype == IRODORI_DTYPE_F32 || dtype == IRODORI_DTYPE_BF16 || dtype == IRODORI_DTYPE_F16;
}
inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// The kernels run on the current device: a stream of another one is refused.  (A null stream is the
// current device's.)  Legal under capture.
inline int check_op_stream(hipStream_t st, const char* op) {
    if (!st) return IRODORI_OK;
    int dev = -1, sdev = -1;
    IRO_HIP_CHECK(hipGetDevice(&dev));
    IRO_HIP_CHECK(hipStreamGetDevice(st, &sdev));
    IRO_REQUIRE(sdev == dev, IRODORI_ERR_INVALID_ARG,
                std::string(op) + ": the stream belongs to device " + std::to_string(sdev) + " but device " +
                    std::to_string(dev) + " is current; make the stream's device current");
    return IRODORI_OK;
}

// Whether the elements of a [n0, n1, n2, inner] tensor with these strides (the inner dimension
// contiguous) all lie at different places, none before the first: what an output needs.
inline bool strides_disjoint(const int64_t (&n)[3], const int64_t* stride, int64_t inner) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
    int64_t extent = inner;
    for (int i : order) {
        if (n[i] == 1) continue;
        if (stride[i] < extent) return false;
        if (stride[i] > (INT64_MAX / 4 - extent) / n[i]) return false;
        extent += stride[i] * (n[i] - 1);
    }
    return true;
}
// Strides that an input may have: none negative (a stride of 0 repeats a row), every offset far inside 64 bits.
inline bool strides_readable(const int64_t (&n)[3], const int64_t* stride) {
    for (int i = 0; i < 3; i++)
        if (n[i] > 1 && (stride[i] < 0 || stride[i] > INT64_MAX / 16 / n[i])) return false;
    return true;
}

}  // namespace irodori
