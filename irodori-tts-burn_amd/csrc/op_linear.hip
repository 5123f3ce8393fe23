// The linear operator's entry points (irodori_op_linear): argument checks and the kernel by type.
#include "common.hpp"
#include "linear.hpp"
#include "op_util.hpp"

using namespace irodori;

namespace {

int check_linear(const irodori_linear_desc* dp) {
    IRO_REQUIRE(dp, IRODORI_ERR_INVALID_ARG, "irodori_op_linear: null description");
    const irodori_linear_desc& d = *dp;
    IRO_REQUIRE(op_dtype_ok(d.dtype), IRODORI_ERR_DTYPE, "irodori_op_linear: dtype must be F32, BF16 or F16");
    IRO_REQUIRE(d.out_dtype == d.dtype || d.out_dtype == IRODORI_DTYPE_F32, IRODORI_ERR_DTYPE,
                "irodori_op_linear: out_dtype must be dtype or F32");
    IRO_REQUIRE(d.m > 0 && d.n > 0 && d.k > 0, IRODORI_ERR_SHAPE, "irodori_op_linear: dims must be positive");
    IRO_REQUIRE(d.m <= 1 << 28 && d.n <= 1 << 28 && d.k <= 1 << 28, IRODORI_ERR_SHAPE,
                "irodori_op_linear: dims must be at most 2^28");
    IRO_REQUIRE(d.activation >= IRODORI_ACT_NONE && d.activation <= IRODORI_ACT_GELU_TANH, IRODORI_ERR_CONFIG,
                "irodori_op_linear: unknown activation");
    IRO_REQUIRE(d.ldx >= 0 && d.ldw >= d.k && d.ldy >= d.n && d.ldr >= 0, IRODORI_ERR_SHAPE,
                "irodori_op_linear: ldw must be at least k, ldy at least n, ldx and ldr not negative");
    const int64_t most = (int64_t)1 << 32;
    IRO_REQUIRE(d.ldx <= most && d.ldw <= most && d.ldy <= most && d.ldr <= most, IRODORI_ERR_SHAPE,
                "irodori_op_linear: a row stride above 2^32");
    IRO_REQUIRE(d.gate_rows >= 0, IRODORI_ERR_SHAPE, "irodori_op_linear: gate_rows must not be negative");
    return IRODORI_OK;
}

// y over something that is read (it may be the residual itself).
bool y_overlaps(const irodori_linear_desc& d, const LinearArgs& a) {
    const size_t es = dtype_bytes(d.dtype), eo = dtype_bytes(d.out_dtype);
    const int64_t nm[3] = {d.m, 1, 1}, nn[3] = {d.n, 1, 1}, sx[3] = {d.ldx}, sw[3] = {d.ldw}, sy[3] = {d.ldy}, sr[3] = {d.ldr};
    const Box y(a.y, eo, nm, sy, d.n), x(a.x, es, nm, sx, d.k), w(a.w, es, nn, sw, d.k), r(a.residual, eo, nm, sr, d.n);
    const Box bias(a.bias, (int64_t)4 * d.n), gate(a.gate, a.gate ? ((int64_t)d.m + d.gate_rows - 1) / d.gate_rows * d.n * 4 : 0);
    return overlap(y, x) || overlap(y, w) || (a.residual != a.y && overlap(y, r)) || overlap(y, bias) || overlap(y, gate);
}

}  // namespace

extern "C" {

int irodori_op_linear_workspace(const irodori_linear_desc* desc, uint64_t* bytes) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_linear(desc));
    IRO_REQUIRE(bytes, IRODORI_ERR_INVALID_ARG, "irodori_op_linear_workspace: null argument");
    *bytes = 0;
    return IRODORI_OK;
    IRO_GUARD_END
}

int irodori_op_linear(const irodori_linear_desc* desc, const void* x, const void* w, const float* bias, const float* gate,
                      const void* residual, void* y, void* workspace, uint64_t workspace_bytes, void* stream) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_linear(desc));
    const irodori_linear_desc& d = *desc;
    IRO_REQUIRE(x && w && y, IRODORI_ERR_INVALID_ARG, "irodori_op_linear: null argument");
    const size_t es = dtype_bytes(d.dtype), eo = dtype_bytes(d.out_dtype);
    IRO_REQUIRE(aligned_to(x, es) && aligned_to(w, es) && aligned_to(y, eo) && aligned_to(residual, eo) &&
                    aligned_to(bias, 4) && aligned_to(gate, 4),
                IRODORI_ERR_INVALID_ARG, "irodori_op_linear: an argument is not aligned to its element type");
    IRO_REQUIRE(!gate == !d.gate_rows, IRODORI_ERR_INVALID_ARG,
                "irodori_op_linear: a gate and a positive gate_rows go together");
    IRO_REQUIRE(y != x && y != w, IRODORI_ERR_INVALID_ARG, "irodori_op_linear: y is an input");
    IRO_REQUIRE(residual != y || d.m == 1 || d.ldr == d.ldy, IRODORI_ERR_SHAPE,
                "irodori_op_linear: y onto its residual needs ldr == ldy");
    hipStream_t st = static_cast<hipStream_t>(stream);
    IRO_TRY(check_op_stream(st, "irodori_op_linear"));
    const LinearArgs a{x, w, residual, y, bias, gate, d.ldx, d.ldw, d.ldy, d.ldr, d.m, d.n, d.k, d.activation, d.gate_rows};
    auto launch = [&](bool go) {
        if (d.dtype == IRODORI_DTYPE_F32) return launch_linear<float, float>(a, st, go);
        if (d.dtype == IRODORI_DTYPE_BF16)
            return d.out_dtype == IRODORI_DTYPE_F32 ? launch_linear<bf16, float>(a, st, go) : launch_linear<bf16, bf16>(a, st, go);
        return d.out_dtype == IRODORI_DTYPE_F32 ? launch_linear<f16, float>(a, st, go) : launch_linear<f16, f16>(a, st, go);
    };
    const bool apart = !y_overlaps(d, a);
    IRO_REQUIRE(launch(apart) == 0, IRODORI_ERR_SHAPE, "irodori_op_linear: too many tiles for one launch");
    IRO_REQUIRE(apart, IRODORI_ERR_INVALID_ARG, "irodori_op_linear: y overlaps an input");
    return check_launch("linear");
    IRO_GUARD_END
}

}  // extern "C"
