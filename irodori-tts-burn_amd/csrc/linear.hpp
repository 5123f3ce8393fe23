// The linear operator's arguments (op_linear.hip checks them, kernels_linear.hip computes).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/irodori_hip.h"

namespace irodori {

struct LinearArgs {
    const void *x, *w, *residual;  // [M, K] and [N, K] in the operand type, [M, N] in the output type
    void* y;                       // [M, N]
    const float *bias, *gate;      // [N]; [ceil(M / gate_rows), N]
    int64_t ldx, ldw, ldy, ldr;    // elements between rows
    int M, N, K, act, gate_rows;
};

// 0, or -1 where the grid would not fit one launch (2^32 threads).  go: false only answers.
template <typename T, typename TO>
int launch_linear(const LinearArgs& a, hipStream_t st, bool go);

}  // namespace irodori
