// The fp8 linear operator's entry point (irodori_op_linear_fp8): argument checks and the kernel by output type.
#include "common.hpp"
#include "fp8_block.hpp"
#include "linear_fp8.hpp"
#include "op_util.hpp"

using namespace irodori;

namespace {

int check_linear_fp8(const irodori_linear_fp8_desc* dp) {
    IRO_REQUIRE(dp, IRODORI_ERR_INVALID_ARG, "irodori_op_linear_fp8: null description");
    const irodori_linear_fp8_desc& d = *dp;
    IRO_REQUIRE(op_dtype_ok(d.out_dtype), IRODORI_ERR_DTYPE, "irodori_op_linear_fp8: out_dtype must be F32, BF16 or F16");
    IRO_REQUIRE(d.m > 0 && d.n > 0 && d.k > 0, IRODORI_ERR_SHAPE, "irodori_op_linear_fp8: dims must be positive");
    IRO_REQUIRE(d.m <= 1 << 28 && d.n <= 1 << 28 && d.k <= 1 << 28, IRODORI_ERR_SHAPE,
                "irodori_op_linear_fp8: dims must be at most 2^28");
    IRO_REQUIRE(d.activation >= IRODORI_ACT_NONE && d.activation <= IRODORI_ACT_GELU_TANH, IRODORI_ERR_CONFIG,
                "irodori_op_linear_fp8: unknown activation");
    IRO_REQUIRE(d.ldx >= 0 && d.ldw >= d.k && d.ldy >= d.n && d.ldr >= 0, IRODORI_ERR_SHAPE,
                "irodori_op_linear_fp8: ldw must be at least k, ldy at least n, ldx and ldr not negative");
    IRO_REQUIRE(d.ldxs >= 0 && d.ldws >= 0, IRODORI_ERR_SHAPE, "irodori_op_linear_fp8: ldxs and ldws must not be negative");
    const int64_t most = (int64_t)1 << 32;
    for (int64_t ld : {d.ldx, d.ldw, d.ldy, d.ldr, d.ldxs, d.ldws})
        IRO_REQUIRE(ld <= most, IRODORI_ERR_SHAPE, "irodori_op_linear_fp8: a row stride above 2^32");
    IRO_REQUIRE(d.gate_rows >= 0, IRODORI_ERR_SHAPE, "irodori_op_linear_fp8: gate_rows must not be negative");
    return IRODORI_OK;
}

// y over something that is read (it may be the residual itself).
bool y_overlaps(const irodori_linear_fp8_desc& d, const LinearFp8Args& a) {
    const size_t eo = dtype_bytes(d.out_dtype);
    const int64_t nm[3] = {d.m, 1, 1}, nn[3] = {d.n, 1, 1}, nb[3] = {((int64_t)d.n + kBlock - 1) / kBlock, 1, 1};
    const int64_t sx[3] = {d.ldx}, sw[3] = {d.ldw}, sy[3] = {d.ldy}, sr[3] = {d.ldr}, sxs[3] = {d.ldxs}, sws[3] = {d.ldws};
    const Box y(a.l.y, eo, nm, sy, d.n), r(a.l.residual, eo, nm, sr, d.n);
    const Box in[] = {Box(a.l.x, 1, nm, sx, d.k), Box(a.l.w, 1, nn, sw, d.k), Box(a.xs, 4, nm, sxs, a.blocks), Box(a.ws, 4, nb, sws, a.blocks),
                      Box(a.l.bias, (int64_t)4 * d.n),
                      Box(a.l.gate, a.l.gate ? ((int64_t)d.m + d.gate_rows - 1) / d.gate_rows * d.n * 4 : 0)};
    for (const Box& b : in)
        if (overlap(y, b)) return true;
    return a.l.residual != a.l.y && overlap(y, r);
}

}  // namespace

extern "C" {

int irodori_op_linear_fp8(const irodori_linear_fp8_desc* desc, const uint8_t* x, const float* x_scales, const uint8_t* w,
                          const float* w_scales, const float* bias, const float* gate, const void* residual, void* y, void* stream) {
    IRO_GUARD_BEGIN
    IRO_TRY(check_linear_fp8(desc));
    const irodori_linear_fp8_desc& d = *desc;
    IRO_REQUIRE(x && x_scales && w && w_scales && y, IRODORI_ERR_INVALID_ARG, "irodori_op_linear_fp8: null argument");
    const size_t eo = dtype_bytes(d.out_dtype);
    IRO_REQUIRE(aligned_to(y, eo) && aligned_to(residual, eo) && aligned_to(x_scales, 4) && aligned_to(w_scales, 4) &&
                    aligned_to(bias, 4) && aligned_to(gate, 4),
                IRODORI_ERR_INVALID_ARG, "irodori_op_linear_fp8: an argument is not aligned to its element type");
    IRO_REQUIRE(!gate == !d.gate_rows, IRODORI_ERR_INVALID_ARG,
                "irodori_op_linear_fp8: a gate and a positive gate_rows go together");
    IRO_REQUIRE(residual != y || d.m == 1 || d.ldr == d.ldy, IRODORI_ERR_SHAPE,
                "irodori_op_linear_fp8: y onto its residual needs ldr == ldy");
    hipStream_t st = static_cast<hipStream_t>(stream);
    IRO_TRY(check_op_stream(st, "irodori_op_linear_fp8"));
    const LinearFp8Args a{{x, w, residual, y, bias, gate, d.ldx, d.ldw, d.ldy, d.ldr, d.m, d.n, d.k, d.activation, d.gate_rows},
                          x_scales, w_scales, d.ldxs, d.ldws, blocks_of(d.k)};
    const bool apart = !y_overlaps(d, a);
    int rc;
    if (d.out_dtype == IRODORI_DTYPE_F32) rc = launch_linear_fp8<float>(a, st, apart);
    else if (d.out_dtype == IRODORI_DTYPE_BF16) rc = launch_linear_fp8<bf16>(a, st, apart);
    else rc = launch_linear_fp8<f16>(a, st, apart);
    IRO_REQUIRE(rc == 0, IRODORI_ERR_SHAPE, "irodori_op_linear_fp8: too many tiles for one launch");
    IRO_REQUIRE(apart, IRODORI_ERR_INVALID_ARG, "irodori_op_linear_fp8: y overlaps an input");
    return check_launch("linear fp8");
    IRO_GUARD_END
}

}  // extern "C"
