// The cross-attention operator's entry points (irodori_op_cross_attention and its workspace):
// argument checks and the kernel by type and head width.
#include "common.hpp"
#include "cross_attention.hpp"
#include "op_util.hpp"

using namespace irodori;

namespace {

int check_cross(const irodori_cross_attention_desc* dp) {
    IRO_REQUIRE(dp, IRODORI_ERR_INVALID_ARG, "irodori_op_cross_attention: null description");
    const irodori_cross_attention_desc& d = *dp;
    IRO_REQUIRE(op_dtype_ok(d.dtype), IRODORI_ERR_DTYPE, "irodori_op_cross_attention: dtype must be F32, BF16 or F16");
    IRO_REQUIRE(d.batch > 0 && d.seq_q > 0 && d.seq_kv > 0 && d.heads > 0 && d.kv_heads > 0, IRODORI_ERR_SHAPE,
                "irodori_op_cross_attention: dims must be positive");
    IRO_REQUIRE(d.head_dim == 64 || d.head_dim == 128, IRODORI_ERR_SHAPE,
                "irodori_op_cross_attention: head_dim must be 64 or 128");
    IRO_REQUIRE(d.heads % d.kv_heads == 0, IRODORI_ERR_SHAPE, "irodori_op_cross_attention: heads must be a multiple of kv_heads");
    IRO_REQUIRE((int64_t)d.seq_q * (d.heads / d.kv_heads) <= 1 << 28 && d.seq_kv <= 1 << 29, IRODORI_ERR_SHAPE,
                "irodori_op_cross_attention: more than 2^28 rows of a key head or 2^29 keys");
    IRO_REQUIRE(std::fabs(d.scale) <= 1e38f, IRODORI_ERR_CONFIG, "irodori_op_cross_attention: scale must be at most 1e38 in magnitude");
    const int64_t qn[3] = {d.batch, d.seq_q, d.heads}, kn[3] = {d.batch, d.seq_kv, d.kv_heads};
    IRO_REQUIRE(strides_readable(qn, d.q_strides) && strides_readable(kn, d.k_strides) && strides_readable(kn, d.v_strides),
                IRODORI_ERR_SHAPE, "irodori_op_cross_attention: a negative or too large stride");
    IRO_REQUIRE(strides_disjoint(qn, d.out_strides, d.head_dim), IRODORI_ERR_SHAPE,
                "irodori_op_cross_attention: the strides of out let its elements overlap");
    IRO_REQUIRE(d.mask_stride >= 0, IRODORI_ERR_SHAPE, "irodori_op_cross_attention: mask_stride must not be negative");
    return IRODORI_OK;
}

int splits_of(const irodori_cross_attention_desc& d) {
    return cross_splits(d.dtype == IRODORI_DTYPE_F32, d.batch, d.kv_heads, d.seq_q * (d.heads / d.kv_heads), d.seq_kv,
                        d.head_dim);
}
int64_t bytes_of(const irodori_cross_attention_desc& d, int splits) {
    return cross_partial_bytes(splits, d.batch, d.kv_heads, d.seq_q * (d.heads / d.kv_heads), d.head_dim);
}

template <typename T>
int run(const CrossArgs& a, int head_dim, hipStream_t st, bool go) {
    return head_dim == 64 ? launch_cross<T, 64>(a, st, go) : launch_cross<T, 128>(a, st, go);
}

// out or the workspace over something that is read, or over one another.
bool outputs_overlap(const irodori_cross_attention_desc& d, const CrossArgs& a, int64_t workspace) {
    const size_t es = dtype_bytes(d.dtype);
    const int64_t nq[3] = {d.batch, d.seq_q, d.heads}, nk[3] = {d.batch, d.seq_kv, d.kv_heads}, nm[3] = {d.batch, 1, 1},
                  sm[3] = {d.mask_stride};
    const Box out(a.out, es, nq, d.out_strides, d.head_dim), ws(workspace ? a.partial : nullptr, workspace);
    const Box in[] = {Box(a.q, es, nq, d.q_strides, d.head_dim), Box(a.k, es, nk, d.k_strides, d.head_dim),
                      Box(a.v, es, nk, d.v_strides, d.head_dim), Box(a.mask, 1, nm, sm, d.seq_kv),
                      Box(a.q_len, (int64_t)4 * d.batch), Box(a.kv_len, (int64_t)4 * d.batch)};
    for (const Box& x : in)
        if (overlap(out, x) || overlap(ws, x)) return true;
    return overlap(out, ws);
}

}  // namespace

extern "C" {

int irodori_op_cross_attention_workspace(const irodori_cross_attention_desc* desc, uint64_t* bytes) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_cross(desc));
    IRO_REQUIRE(bytes, IRODORI_ERR_INVALID_ARG, "irodori_op_cross_attention_workspace: null argument");
    *bytes = (uint64_t)bytes_of(*desc, splits_of(*desc));
    return IRODORI_OK;
    IRO_GUARD_END
}

int irodori_op_cross_attention(const irodori_cross_attention_desc* desc, const void* q, const void* k, const void* v,
                               const uint8_t* mask, const int32_t* q_len, const int32_t* kv_len, void* out,
                               void* workspace, uint64_t workspace_bytes, void* stream) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_cross(desc));
    const irodori_cross_attention_desc& d = *desc;
    IRO_REQUIRE(q && k && v && out, IRODORI_ERR_INVALID_ARG, "irodori_op_cross_attention: null argument");
    const size_t es = dtype_bytes(d.dtype);
    IRO_REQUIRE(aligned_to(q, es) && aligned_to(k, es) && aligned_to(v, es) && aligned_to(out, es) &&
                    aligned_to(q_len, 4) && aligned_to(kv_len, 4),
                IRODORI_ERR_INVALID_ARG, "irodori_op_cross_attention: an argument is not aligned to its element type");
    const int splits = splits_of(d);
    const int64_t need = bytes_of(d, splits);
    IRO_REQUIRE(need == 0 || (workspace && workspace_bytes >= (uint64_t)need && aligned_to(workspace, 16)), IRODORI_ERR_INVALID_ARG,
                "irodori_op_cross_attention: this shape takes a 16-byte aligned workspace of " + std::to_string(need) + " bytes");
    IRO_REQUIRE(out != q && out != k && out != v, IRODORI_ERR_INVALID_ARG, "irodori_op_cross_attention: out is an input");
    hipStream_t st = static_cast<hipStream_t>(stream);
    IRO_TRY(check_op_stream(st, "irodori_op_cross_attention"));
    CrossArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.mask = mask; a.q_len = q_len; a.kv_len = kv_len;
    a.partial = static_cast<float*>(workspace);
    const int qn[3] = {d.batch, d.seq_q, d.heads}, kn[3] = {d.batch, d.seq_kv, d.kv_heads};
    for (int i = 0; i < 3; i++) {  // (the stride of a dimension of one says nothing)
        a.qs[i] = qn[i] > 1 ? d.q_strides[i] : 0; a.os[i] = qn[i] > 1 ? d.out_strides[i] : 0;
        a.ks[i] = kn[i] > 1 ? d.k_strides[i] : 0; a.vs[i] = kn[i] > 1 ? d.v_strides[i] : 0;
    }
    // A tile's rows past a single key lie behind it, outside its window: at stride 0 each would read as that key, and
    // a weight of 0 times an infinite value is not 0.
    if (d.seq_kv == 1) a.ks[1] = a.vs[1] = d.head_dim;
    a.mask_stride = d.mask_stride;
    a.batch = d.batch; a.heads = d.heads; a.kv_heads = d.kv_heads; a.group = d.heads / d.kv_heads;
    a.seq_q = d.seq_q; a.seq_kv = d.seq_kv; a.splits = splits;
    a.rows = d.seq_q * a.group;
    a.scale = d.scale;
    const bool apart = !outputs_overlap(d, a, need);
    int rc;
    if (d.dtype == IRODORI_DTYPE_BF16) rc = run<bf16>(a, d.head_dim, st, apart);
    else if (d.dtype == IRODORI_DTYPE_F16) rc = run<f16>(a, d.head_dim, st, apart);
    else rc = run<float>(a, d.head_dim, st, apart);
    IRO_REQUIRE(rc == 0, IRODORI_ERR_SHAPE, "irodori_op_cross_attention: too many rows for one launch");
    IRO_REQUIRE(apart, IRODORI_ERR_INVALID_ARG, "irodori_op_cross_attention: out or the workspace overlaps another argument");
    return check_launch("cross attention");
    IRO_GUARD_END
}

}  // extern "C"
