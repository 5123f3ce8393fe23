"""What the operators of an fp8 half block (irodori_op_block_norm, irodori_op_block_quantize,
irodori_op_linear_fp8) refuse, through the C ABI without a device: every call here fails before its first
device call."""
import ctypes as C

import pytest

import irodori_hip as ih
from irodori_hip import _lib as L
from irodori_hip.config import IrodoriError

M = 1 << 24  # addresses this far apart, which no refused call reads


def norm_desc(**kw):
    base = dict(rows=6, dim=256)
    base.update(kw)
    return ih.BlockNormDesc(base.pop("rows"), base.pop("dim"), **base)


def quant_desc(**kw):
    base = dict(rows=6, dim=256)
    base.update(kw)
    return ih.BlockQuantizeDesc(base.pop("rows"), base.pop("dim"), **base)


def linear_desc(**kw):
    base = dict(m=6, n=256, k=300)
    base.update(kw)
    return ih.LinearFp8Desc(base.pop("m"), base.pop("n"), base.pop("k"), **base)


def norm_args(*names, **at):
    """Every tensor of the names (x and h always) at a place of its own, `at` instead of it."""
    order = ("x", "h", "branch", "branch_weight", "branch_bias", "gate", "x_out", "weight", "bias", "scale", "shift", "h_scales")
    args = {"d_" + n: M * (1 + i) for i, n in enumerate(order) if n in names + ("x", "h")}
    args.update({"d_" + n: p for n, p in at.items()})
    return args


def norm(desc, *names, **at):
    return lambda: ih.ops.block_norm(desc, **norm_args(*names, **at))


def quant(desc, x=M, q=2 * M, s=3 * M):
    return lambda: ih.ops.block_quantize(desc, x, q, s)


def linear(desc, **at):
    args = dict(d_x=M, d_x_scales=2 * M, d_w=3 * M, d_w_scales=4 * M, d_y=5 * M)
    args.update(at)
    return lambda: ih.ops.linear_fp8(desc, **args)


def edited(desc, **fields):
    for name, value in fields.items():
        setattr(desc, name, value)
    return desc


def refused(kind, text, call):
    with pytest.raises(IrodoriError) as e:
        call()
    assert e.value.kind == kind and text in str(e.value), str(e.value)


def test_description_sizes_match_the_header():
    assert C.sizeof(L.BlockNormDescC) == 8 * 4 + 4 * 4 + 6 * 8
    assert C.sizeof(L.BlockQuantizeDescC) == 6 * 4 + 3 * 8
    assert C.sizeof(L.LinearFp8DescC) == 6 * 4 + 6 * 8


@pytest.mark.parametrize("kw,kind,text", [
    (dict(rows=0), "Shape", "positive"), (dict(dim=0), "Shape", "positive"), (dict(rows=-1), "Shape", "positive"),
    (dict(dim=16385), "Shape", "16384"), (dict(eps=0.0), "Config", "eps"), (dict(branch_eps=float("nan")), "Config", "eps"),
    (dict(eps=1e31), "Config", "eps"), (dict(stream_scale=float("inf")), "Config", "scales"),
    (dict(branch_scale=float("nan")), "Config", "scales"), (dict(mod_rows=-1), "Shape", "mod_rows"),
    (dict(ldx=-1), "Shape", "ldx"), (dict(ldb=-1), "Shape", "ldb"), (dict(ldxo=255), "Shape", "ldxo"), (dict(ldh=255), "Shape", "ldh"),
    (dict(ldhs=1), "Shape", "ldhs"), (dict(ldm=-1), "Shape", "ldm"), (dict(ldx=2 ** 33), "Shape", "2^32"),
    (dict(dtype="bf16", stream_dtype="f16"), "Dtype", "stream_dtype"), (dict(dtype="bf16", h_dtype="f32"), "Dtype", "h_dtype"),
])
def test_block_norm_refusals(kw, kind, text):
    refused(kind, text, norm(norm_desc(**kw), "x_out"))


def test_block_norm_refuses_pointers_and_codes():
    d = norm_desc()
    refused("InvalidArg", "null", norm(d, x=0))
    refused("InvalidArg", "null", norm(d, h=0))
    for n in ("branch_weight", "branch_bias"):
        refused("InvalidArg", "without a branch", norm(d, n))
    refused("InvalidArg", "without a branch", norm(norm_desc(mod_rows=2), "gate"))
    for n in ("weight", "bias"):
        refused("InvalidArg", "without h", norm(d, "x_out", n, h=0))
    refused("InvalidArg", "without h", norm(norm_desc(mod_rows=2), "x_out", "scale", h=0))
    refused("InvalidArg", "h_scales", norm(d, "h_scales"))
    refused("InvalidArg", "h_scales", norm(norm_desc(h_dtype="fp8")))
    refused("InvalidArg", "h_scales", norm(norm_desc(h_dtype="fp8"), "x_out", "h_scales", h=0))
    for n in ("scale", "shift"):
        refused("InvalidArg", "mod_rows", norm(d, n))
    refused("InvalidArg", "mod_rows", norm(d, "branch", "gate"))
    refused("InvalidArg", "mod_rows", norm(norm_desc(mod_rows=2), "branch"))
    for n in ("x", "h", "branch", "x_out"):
        refused("InvalidArg", "aligned", norm(d, "branch", "x_out", **{n: 20 * M + 1}))
    for n in ("branch_weight", "branch_bias", "gate", "weight", "bias", "scale", "shift"):
        refused("InvalidArg", "aligned", norm(norm_desc(mod_rows=2), "branch", "gate", **{n: 20 * M + 2}))
    refused("InvalidArg", "aligned", norm(norm_desc(h_dtype="fp8"), h_scales=20 * M + 2))
    refused("Shape", "in place", norm(norm_desc(ldx=300), "x_out", x_out=M))
    refused("Dtype", "dtype", norm(edited(norm_desc(), dtype=L.DTYPE_FP8)))
    refused("Config", "norm", norm(edited(norm_desc(), norm=3)))
    refused("Config", "norm", norm(edited(norm_desc(), branch_norm=-1)))
    assert L.load().irodori_op_block_norm(None, *[M] * 12, None) == L.ERR_INVALID_ARG
    for kw in (dict(dtype="fp8"), dict(stream_dtype="fp8"), dict(h_dtype="fp4"), dict(norm="batch"), dict(branch_norm="l2")):
        refused("Config", "must be one of", lambda: norm_desc(**kw))


def test_block_norm_refuses_outputs_over_other_arguments():
    names = ("branch", "branch_weight", "branch_bias", "gate", "x_out", "weight", "bias", "scale", "shift", "h_scales")
    d = norm_desc(h_dtype="fp8", mod_rows=4)
    place = norm_args(*names)
    for out in ("x_out", "h", "h_scales"):
        for other in ("x", "h") + names:
            if other == out:
                continue
            refused("InvalidArg", "overlaps", norm(d, *names, **{out: place["d_" + other] + 4}))
            if (out, other) != ("x_out", "x"):
                refused("InvalidArg", "overlaps", norm(d, *names, **{out: place["d_" + other]}))
    # The last of the modulation's rows.
    refused("InvalidArg", "overlaps", norm(norm_desc(h_dtype="fp8", mod_rows=4, ldm=700), *names, x_out=place["d_gate"] + 4 * 700))


@pytest.mark.parametrize("kw,kind,text", [
    (dict(rows=0), "Shape", "positive"), (dict(dim=-5), "Shape", "positive"), (dict(rows=2 ** 28 + 1), "Shape", "2^28"),
    (dict(block_rows=2), "Config", "block_rows"), (dict(block_rows=0), "Config", "block_rows"),
    (dict(block_rows=128, gated=True), "Config", "activation"), (dict(block_rows=128, activation="silu"), "Config", "activation"),
    (dict(ldx=-1), "Shape", "ldx"), (dict(ldq=255), "Shape", "ldq"), (dict(lds=1), "Shape", "lds"), (dict(ldq=2 ** 33), "Shape", "2^32"),
])
def test_block_quantize_refusals(kw, kind, text):
    refused(kind, text, quant(quant_desc(**kw)))


def test_block_quantize_refuses_pointers_and_codes():
    d = quant_desc()
    for kw in (dict(x=0), dict(q=0), dict(s=0)):
        refused("InvalidArg", "null", quant(d, **kw))
    refused("InvalidArg", "aligned", quant(d, x=M + 1))
    refused("InvalidArg", "aligned", quant(d, s=M + 2))
    refused("Dtype", "dtype", quant(edited(quant_desc(), dtype=L.DTYPE_FP8)))
    refused("Config", "activation", quant(edited(quant_desc(), activation=7)))
    assert L.load().irodori_op_block_quantize(None, M, M, M, None) == L.ERR_INVALID_ARG
    row = 256 * 2
    for kw in (dict(q=M), dict(q=M + 5 * row + row - 1), dict(s=M + 8), dict(s=2 * M + 4), dict(s=2 * M - 4 * 11)):
        refused("InvalidArg", "overlaps", quant(d, **kw))
    # the second half of a gated row
    refused("InvalidArg", "overlaps", quant(quant_desc(gated=True), q=M + 6 * 2 * row - 1))


@pytest.mark.parametrize("kw,kind,text", [
    (dict(m=0), "Shape", "positive"), (dict(n=0), "Shape", "positive"), (dict(k=-1), "Shape", "positive"),
    (dict(k=2 ** 28 + 1), "Shape", "2^28"), (dict(ldw=299), "Shape", "ldw"), (dict(ldy=255), "Shape", "ldy"),
    (dict(ldx=-1), "Shape", "ldx"), (dict(ldr=-1), "Shape", "ldr"), (dict(ldxs=-1), "Shape", "ldxs"), (dict(ldws=-1), "Shape", "ldws"),
    (dict(ldws=2 ** 33), "Shape", "2^32"), (dict(gate_rows=-1), "Shape", "gate_rows"),
])
def test_linear_fp8_refusals(kw, kind, text):
    refused(kind, text, linear(linear_desc(**kw)))


def test_linear_fp8_refuses_pointers_and_codes():
    d = linear_desc()
    for n in ("d_x", "d_x_scales", "d_w", "d_w_scales", "d_y"):
        refused("InvalidArg", "null", linear(d, **{n: 0}))
    for kw in (dict(d_x_scales=M + 1), dict(d_w_scales=M + 2), dict(d_y=9 * M + 1), dict(d_bias=M + 2), dict(d_residual=M + 1)):
        refused("InvalidArg", "aligned", linear(d, **kw))
    refused("InvalidArg", "aligned", linear(linear_desc(gate_rows=2), d_gate=M + 2))
    refused("InvalidArg", "gate_rows", linear(d, d_gate=M))
    refused("InvalidArg", "gate_rows", linear(linear_desc(gate_rows=2)))
    refused("Shape", "ldr", linear(linear_desc(ldr=257), d_residual=5 * M))
    refused("Config", "activation", linear(edited(linear_desc(), activation=7)))
    refused("Dtype", "out_dtype", linear(edited(linear_desc(), out_dtype=L.DTYPE_FP8)))
    refused("Config", "must be one of", lambda: linear_desc(out_dtype="fp8"))
    assert L.load().irodori_op_linear_fp8(None, *[M] * 8, None) == L.ERR_INVALID_ARG


def test_linear_fp8_refuses_outputs_over_other_arguments():
    d = linear_desc(gate_rows=2)
    place = dict(d_x=M, d_x_scales=2 * M, d_w=3 * M, d_w_scales=4 * M, d_bias=6 * M, d_gate=7 * M, d_residual=8 * M)
    for n in place:
        refused("InvalidArg", "overlaps", linear(d, **dict(place, d_y=place[n] + 2)))
    for n in ("d_x", "d_w", "d_x_scales", "d_w_scales", "d_bias", "d_gate"):
        refused("InvalidArg", "overlaps", linear(d, **dict(place, d_y=place[n])))
    # the last row of each
    for n, at in (("d_x", 5 * 300), ("d_x_scales", 4 * 5 * 3), ("d_w", 255 * 300), ("d_w_scales", 4 * 3), ("d_gate", 4 * 2 * 256)):
        refused("InvalidArg", "overlaps", linear(d, **dict(place, d_y=place[n] + at)))


@pytest.mark.parametrize("text,call", [
    ("rows", norm(norm_desc(rows=2 ** 26, dim=64, ldx=64))),
    ("rows", norm(norm_desc(rows=2 ** 24, dim=16384))),
    ("blocks", lambda: ih.ops.block_quantize(quant_desc(rows=2 ** 28, dim=640), M, 2 ** 44, 2 ** 45)),
    ("blocks", lambda: ih.ops.block_quantize(quant_desc(rows=2 ** 28, dim=2 ** 14, block_rows=128), M, 2 ** 46, 2 ** 47)),
    ("tiles", linear(linear_desc(m=1, n=2 ** 28, k=1))),
    ("tiles", linear(linear_desc(m=2 ** 28, n=2 ** 28, k=1))),
])
def test_more_work_than_a_launch_holds_is_refused(text, call):
    # A launch has at most 2^32 - 1 threads in one dimension.
    refused("Shape", text + " for one launch", call)


def test_numbers_that_the_fields_cannot_hold_are_refused():
    for text, make in (("rows of", lambda: norm_desc(rows=2 ** 32 + 4)), ("dim of", lambda: norm_desc(dim=-2 ** 32 + 16)),
                       ("ldm of", lambda: norm_desc(ldm=2 ** 64 + 16)), ("dim of", lambda: quant_desc(dim=2 ** 32 + 7)),
                       ("block_rows of", lambda: quant_desc(block_rows=2 ** 32 + 1)), ("ldq of", lambda: quant_desc(ldq=2 ** 63)),
                       ("k of", lambda: linear_desc(k=2 ** 32 + 128)), ("ldxs of", lambda: linear_desc(ldxs=2 ** 64))):
        refused("Shape", text, make)
