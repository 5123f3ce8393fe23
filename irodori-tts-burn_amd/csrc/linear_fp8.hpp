// The fp8 linear operator's arguments (op_linear_fp8.hip checks them, kernels_linear_fp8.hip computes).
#pragma once

#include "linear.hpp"

namespace irodori {

struct LinearFp8Args {
    LinearArgs l;           // x and w: e4m3 codes
    const float *xs, *ws;   // scales [M, blocks] and [ceil(N / 128), blocks] of 128 codes along K
    int64_t ldxs, ldws;     // elements between their rows
    int blocks;
};

// 0, or -1 where the grid would not fit one launch (2^32 threads).  go: false only answers.
template <typename TO>
int launch_linear_fp8(const LinearFp8Args& a, hipStream_t st, bool go);

}  // namespace irodori
