// The cross-attention operator's arguments (op_cross_attention.hip checks them,
// kernels_cross_attention.hip computes).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace irodori {

struct CrossArgs {
    const void *q, *k, *v;
    void* out;
    const uint8_t* mask;          // [batch][mask_stride], nonzero = attend; may be null
    const int32_t *q_len, *kv_len;  // [batch]; may be null
    float* partial;               // splits > 1: [kv_heads][splits + batch][rows][head_dim], then (m, l) of each row
    int64_t qs[3], ks[3], vs[3], os[3];  // batch, token, head strides in elements
    int64_t mask_stride;
    int batch, heads, kv_heads, group, seq_q, seq_kv, splits;
    int rows;  // seq_q * group: row r is token r / group of head r % group of the kv head's group
    float scale;
};

// Runs that the keys of a launch are split into (1: none), and the bytes of their partial results.
int cross_splits(bool f32, int batch, int kv_heads, int rows, int seq_kv, int head_dim);
inline int64_t cross_partial_bytes(int splits, int batch, int kv_heads, int rows, int head_dim) {
    return splits > 1 ? ((int64_t)splits + batch) * kv_heads * rows * (head_dim + 2) * 4 : 0;
}

// 0, or -1 where the grid would not fit one launch (2^32 threads).  go: false only answers.
template <typename T, int DH>
int launch_cross(const CrossArgs& a, hipStream_t st, bool go);

}  // namespace irodori
