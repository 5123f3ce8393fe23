// Host checks and device element helpers shared by the described operators (op_rope.hip,
// op_linear.hip, op_cross_attention.hip, op_block_norm.hip, op_block_quantize.hip, op_linear_fp8.hip).
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

// The bytes of a tensor: n[0] x n[1] x n[2] rows of `inner` bytes, strides in bytes.  (128-bit sums: any stride that the
// checks above let through.)
typedef __int128 wide_t;
struct Box {
    wide_t at, n[3], stride[3], inner;
    Box(const void* p, size_t element, const int64_t (&dims)[3], const int64_t* strides, int64_t row)
        : at(reinterpret_cast<uintptr_t>(p)), inner((wide_t)row * element) {
        for (int i = 0; i < 3; i++) {
            n[i] = dims[i];
            stride[i] = n[i] > 1 ? (wide_t)strides[i] * element : 0;
        }
    }
    Box(const void* p, int64_t bytes) : at(reinterpret_cast<uintptr_t>(p)), n{1, 1, 1}, stride{0, 0, 0}, inner(bytes) {}
    wide_t end() const { return at + (n[0] - 1) * stride[0] + (n[1] - 1) * stride[1] + (n[2] - 1) * stride[2] + inner; }
    bool dense() const {  // no byte between its first and its last is left out
        int order[3] = {0, 1, 2};
        std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
        wide_t extent = inner;
        for (int i : order) {
            if (stride[i] > extent) return false;
            extent += (n[i] - 1) * stride[i];
        }
        return true;
    }
};
// Whether two tensors certainly share a byte: where one has no gaps, or where their strides are equal (parts of one
// buffer).  Two with gaps and different strides may do so unseen.
inline bool overlap(const Box& a, const Box& b) {
    if (!a.at || !b.at || a.end() <= b.at || b.end() <= a.at) return false;
    auto meets = [](const Box& x, const Box& y) {  // y's first or last row lies in x, which has no gaps
        return x.dense() && ((y.at < x.end() && x.at < y.at + y.inner) || (y.end() - y.inner < x.end() && x.at < y.end()));
    };
    if (meets(a, b) || meets(b, a)) return true;
    // b.at - a.at = sum of i s over the strides, i between -(b.n - 1) and a.n - 1, and a rest between -(b.inner - 1) and
    // a.inner - 1: the larger strides first, each with the few multiples that leave what the others can make up.
    struct Dim { wide_t s, lo, hi; } dim[3];
    for (int i = 0; i < 3; i++) {
        if (a.n[i] > 1 && b.n[i] > 1 && a.stride[i] != b.stride[i]) return false;
        dim[i] = {a.n[i] > 1 ? a.stride[i] : b.stride[i], 1 - b.n[i], a.n[i] - 1};
    }
    std::sort(dim, dim + 3, [](const Dim& x, const Dim& y) { return x.s > y.s; });
    auto floor_div = [](wide_t x, wide_t y) { return x / y - (x % y < 0); };
    auto reach = [&](auto& self, int k, wide_t d) -> bool {
        wide_t lo = 1 - b.inner, hi = a.inner - 1;  // of dimensions k + 1 and on and the rest
        for (int j = k + 1; j < 3; j++) {
            lo += dim[j].lo * dim[j].s;
            hi += dim[j].hi * dim[j].s;
        }
        if (k == 3 || dim[k].s == 0) return lo <= d && d <= hi;
        const wide_t first = std::max(dim[k].lo, -floor_div(hi - d, dim[k].s)), last = std::min(dim[k].hi, floor_div(d - lo, dim[k].s));
        for (wide_t i = first; i <= last && i < first + 8; i++)
            if (self(self, k + 1, d - i * dim[k].s)) return true;
        return false;
    };
    return reach(reach, 0, b.at - a.at);
}

}  // namespace irodori
