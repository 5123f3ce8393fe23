"""What the described operators (irodori_op_rope, irodori_op_linear, irodori_op_cross_attention)
refuse, through the C ABI without a device: every call here fails, or answers, before its first
device call."""
import ctypes as C
import itertools

import pytest

import irodori_hip as ih
from irodori_hip import _lib as L
from irodori_hip.config import IrodoriError

P = 4096  # an aligned address that no refused call reads


def rope_desc(**kw):
    base = dict(batch=2, seq=5, head_dim=64, heads=4, kv_heads=2)
    base.update(kw)
    return ih.RopeDesc(base.pop("batch"), base.pop("seq"), base.pop("head_dim"), **base)


def linear_desc(**kw):
    base = dict(m=4, n=8, k=16)
    base.update(kw)
    return ih.LinearDesc(base.pop("m"), base.pop("n"), base.pop("k"), **base)


def cross_desc(**kw):
    base = dict(batch=2, seq_q=3, seq_kv=7, heads=4, kv_heads=2, head_dim=64)
    base.update(kw)
    return ih.CrossAttentionDesc(**base)


def edited(desc, **fields):
    for name, value in fields.items():
        setattr(desc, name, value)
    return desc


def refused(kind, text, call):
    with pytest.raises(IrodoriError) as e:
        call()
    assert e.value.kind == kind and text in str(e.value), str(e.value)


def test_description_sizes_match_the_header():
    # Fields as include/irodori_hip.h declares them, naturally aligned.
    assert C.sizeof(L.RopeDescC) == 14 * 4 + 6 * 8 + 12 * 8
    assert C.sizeof(L.LinearDescC) == 8 * 4 + 4 * 8
    assert C.sizeof(L.CrossAttentionDescC) == 8 * 4 + 12 * 8 + 8


@pytest.mark.parametrize("kw,kind,text", [
    (dict(batch=0), "Shape", "positive"), (dict(seq=0), "Shape", "positive"), (dict(seq=-3), "Shape", "positive"),
    (dict(heads=0, kv_heads=0), "Shape", "heads"), (dict(heads=20000), "Shape", "heads"),
    (dict(head_dim=1026, rot_dim=64), "Shape", "head_dim"), (dict(head_dim=63, rot_dim=62), "Shape", "even"),
    (dict(rot_dim=0), "Shape", "rot_dim"), (dict(rot_dim=63), "Shape", "rot_dim"), (dict(rot_dim=66), "Shape", "rot_dim"),
    (dict(head_dim=1024, rot_dim=514), "Shape", "rot_dim"), (dict(rot_heads=5), "Shape", "rot_heads"),
    (dict(rot_kv_heads=-1), "Shape", "rot_heads"), (dict(theta=0.0), "Config", "theta"), (dict(theta=float("nan")), "Config", "theta"),
    (dict(amplitude=float("inf")), "Config", "amplitude"), (dict(amplitude=-1e300), "Config", "amplitude"),
    (dict(scaling="linear", factor=1e-30), "Config", "frequency"), (dict(theta=1e-300), "Config", "frequency"), (dict(scaling="linear", factor=0.0), "Config", "factor"),
    (dict(scaling="ntk", factor=2.0, rot_dim=2), "Config", "rot_dim"),
    (dict(scaling="by_parts", factor=2.0), "Config", "trained_len"),
    (dict(scaling="by_parts", factor=2.0, trained_len=100.0, beta_fast=1.0), "Config", "beta_fast"),
    (dict(first_pos=2 ** 31 - 3), "Shape", "2^31"), (dict(seq=2 ** 30 + 1), "Shape", "2^30"),
    (dict(q_strides=(-1, 256, 64)), "Shape", "stride"), (dict(k_out_strides=(640, 128, 32)), "Shape", "overlap"),
    (dict(q_out_strides=(0, 256, 64)), "Shape", "overlap"),
])
def test_rope_refusals(kw, kind, text):
    refused(kind, text, lambda: ih.ops.rope(rope_desc(**kw), P, 2 * P, 3 * P, 4 * P))


def test_rope_refuses_pointers_and_codes():
    d = rope_desc()
    for args in ((0, P, P, 2 * P), (P, 0, P, 2 * P), (P, 2 * P, 0, P), (P, 2 * P, P, 0)):
        refused("InvalidArg", "null", lambda: ih.ops.rope(d, *args))
    refused("InvalidArg", "aligned", lambda: ih.ops.rope(d, P + 1, 2 * P, 3 * P, 4 * P))
    refused("InvalidArg", "aligned", lambda: ih.ops.rope(d, P, 2 * P, 3 * P, 4 * P, d_positions=P + 2))
    refused("Shape", "in place", lambda: ih.ops.rope(rope_desc(q_strides=(10000, 512, 64)), P, P, 3 * P, 4 * P))
    refused("Dtype", "dtype", lambda: ih.ops.rope(edited(rope_desc(), dtype=L.DTYPE_FP8), P, 2 * P, 3 * P, 4 * P))
    refused("Config", "layout", lambda: ih.ops.rope(edited(rope_desc(), layout=2), P, 2 * P, 3 * P, 4 * P))
    refused("Config", "scaling", lambda: ih.ops.rope(edited(rope_desc(), scaling=4), P, 2 * P, 3 * P, 4 * P))
    assert L.load().irodori_op_rope(None, P, P, P, P, None, None, None) == L.ERR_INVALID_ARG
    for kw in (dict(dtype="fp8"), dict(layout="rows"), dict(scaling="log")):
        refused("Config", "must be one of", lambda: rope_desc(**kw))
    refused("Shape", "strides", lambda: rope_desc(q_strides=(1, 2)))


@pytest.mark.parametrize("kw,kind,text", [
    (dict(m=0), "Shape", "positive"), (dict(n=0), "Shape", "positive"), (dict(k=-1), "Shape", "positive"),
    (dict(m=2 ** 28 + 1), "Shape", "2^28"), (dict(ldw=15), "Shape", "ldw"), (dict(ldy=7), "Shape", "ldy"),
    (dict(ldx=-1), "Shape", "ldx"), (dict(ldr=-1), "Shape", "ldr"), (dict(ldx=2 ** 33), "Shape", "2^32"),
    (dict(gate_rows=-1), "Shape", "gate_rows"), (dict(dtype="bf16", out_dtype="f16"), "Dtype", "out_dtype"),
])
def test_linear_refusals(kw, kind, text):
    refused(kind, text, lambda: ih.ops.linear(linear_desc(**kw), P, 2 * P, 3 * P))


def test_linear_refuses_pointers_and_codes():
    d = linear_desc()
    for args in ((0, P, P), (P, 0, P), (P, P, 0)):
        refused("InvalidArg", "null", lambda: ih.ops.linear(d, *args))
    for kw in (dict(d_bias=P + 2), dict(d_gate=P + 2), dict(d_residual=P + 1)):
        refused("InvalidArg", "aligned", lambda: ih.ops.linear(d, P, 2 * P, 3 * P, **kw))
    refused("InvalidArg", "gate_rows", lambda: ih.ops.linear(d, P, 2 * P, 3 * P, d_gate=P))
    refused("InvalidArg", "gate_rows", lambda: ih.ops.linear(linear_desc(gate_rows=2), P, 2 * P, 3 * P))
    refused("Shape", "ldr", lambda: ih.ops.linear(linear_desc(ldr=9), P, 2 * P, 3 * P, d_residual=3 * P))
    refused("Config", "activation", lambda: ih.ops.linear(edited(linear_desc(), activation=7), P, 2 * P, 3 * P))
    refused("Dtype", "dtype", lambda: ih.ops.linear(edited(linear_desc(), dtype=L.DTYPE_FP8), P, 2 * P, 3 * P))
    refused("Config", "must be one of", lambda: linear_desc(activation="swish"))
    n = C.c_uint64()
    assert L.load().irodori_op_linear_workspace(d, None) == L.ERR_INVALID_ARG
    assert L.load().irodori_op_linear_workspace(None, n) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("kw,kind,text", [
    (dict(batch=0), "Shape", "positive"), (dict(seq_q=0), "Shape", "positive"), (dict(seq_kv=0), "Shape", "positive"),
    (dict(heads=3), "Shape", "multiple"), (dict(kv_heads=0), "Shape", "positive"), (dict(head_dim=96), "Shape", "head_dim"),
    (dict(scale=float("nan")), "Config", "scale"), (dict(scale=-3e38), "Config", "scale"), (dict(seq_q=2 ** 28, heads=4, kv_heads=2), "Shape", "2^28"),
    (dict(seq_kv=2 ** 29 + 1), "Shape", "2^29"), (dict(k_strides=(-64, 128, 64)), "Shape", "stride"),
    (dict(out_strides=(768, 256, 63)), "Shape", "overlap"), (dict(mask_stride=-1), "Shape", "mask_stride"),
])
def test_cross_attention_refusals(kw, kind, text):
    refused(kind, text, lambda: ih.ops.cross_attention(cross_desc(**kw), P, 2 * P, 3 * P, 4 * P))
    refused(kind, text, lambda: ih.ops.cross_attention_workspace(cross_desc(**kw)))


def test_cross_attention_refuses_pointers_and_workspaces():
    d = cross_desc()
    for args in ((0, P, P, P), (P, 0, P, P), (P, P, 0, P), (P, P, P, 0)):
        refused("InvalidArg", "null", lambda: ih.ops.cross_attention(d, *args))
    refused("InvalidArg", "aligned", lambda: ih.ops.cross_attention(d, P, P + 1, P, P))
    refused("InvalidArg", "aligned", lambda: ih.ops.cross_attention(d, P, P, P, P, d_kv_len=P + 2))
    refused("Dtype", "dtype", lambda: ih.ops.cross_attention(edited(cross_desc(), dtype=L.DTYPE_FP8), P, P, P, P))
    # A new token over many keys is split: its workspace is asked for, and has to be there.
    d = cross_desc(batch=1, seq_q=1, seq_kv=100000)
    need = ih.ops.cross_attention_workspace(d)
    assert need > 0
    for kw in (dict(), dict(d_workspace=P, workspace_bytes=need - 1), dict(d_workspace=P + 8, workspace_bytes=need),
               dict(workspace_bytes=need)):
        refused("InvalidArg", "workspace", lambda: ih.ops.cross_attention(d, P, P, P, P, **kw))
    assert L.load().irodori_op_cross_attention_workspace(d, None) == L.ERR_INVALID_ARG


@pytest.mark.parametrize("text,call", [
    ("tokens", lambda: ih.ops.rope(rope_desc(batch=1024, seq=2 ** 30), P, 2 * P, 3 * P, 4 * P)),
    ("tokens", lambda: ih.ops.rope(rope_desc(batch=4096, seq=2 ** 18, dtype="bf16"), P, 2 * P, 3 * P, 4 * P)),
    ("tiles", lambda: ih.ops.linear(linear_desc(m=1, n=2 ** 28, k=1), P, 2 * P, 3 * P)),
    ("tiles", lambda: ih.ops.linear(linear_desc(m=2 ** 28, n=2 ** 28, k=1), P, 2 * P, 3 * P)),
    ("rows", lambda: ih.ops.cross_attention(cross_desc(batch=2 ** 20, seq_q=4096, heads=16, kv_heads=16), P, 2 * P, 3 * P, 4 * P)),
    ("rows", lambda: ih.ops.cross_attention(cross_desc(batch=2 ** 17, seq_q=4096, heads=16, kv_heads=2), P, 2 * P, 3 * P, 4 * P)),
])
def test_more_work_than_a_launch_holds_is_refused(text, call):
    # A launch has at most 2^32 - 1 threads in one dimension.
    refused("Shape", text + " for one launch", call)


def test_outputs_that_are_inputs_are_refused():
    d = cross_desc()
    for at in (P, 2 * P, 3 * P):
        refused("InvalidArg", "out is an input", lambda: ih.ops.cross_attention(d, P, 2 * P, 3 * P, at))
    for at in (P, 2 * P):
        refused("InvalidArg", "y is an input", lambda: ih.ops.linear(linear_desc(), P, 2 * P, at))
    for args in ((P, 2 * P, 3 * P, 2 * P), (P, 3 * P, 3 * P, 4 * P), (P, P, 3 * P, P)):
        refused("InvalidArg", "other side's", lambda: ih.ops.rope(rope_desc(), *args))


def rows(at, dims, strides, inner):
    """The elements of a tensor, as numbers."""
    return {at + sum(i * s for i, s in zip(index, strides)) + e for index in itertools.product(*map(range, dims)) for e in range(inner)}


@pytest.mark.parametrize("heads,between", [(2, 0), (2, 1), (3, 2)])
def test_rope_refuses_outputs_inside_inputs(heads, between):
    # q of one head and the next head's place: every offset inside a buffer of heads that shares an element is refused.
    d, seq, rowlen = 4, 3, (heads + between) * 4
    strides = (seq * rowlen, rowlen, d)
    desc = rope_desc(batch=2, seq=seq, head_dim=d, heads=heads, kv_heads=0, dtype="f32", q_strides=strides, q_out_strides=strides)
    q = rows(0, (2, seq, heads), strides, d)
    seen = 0
    for at in range(-2 * seq * rowlen, 2 * seq * rowlen):
        if at and q & rows(at, (2, seq, heads), strides, d):
            refused("InvalidArg", "overlaps", lambda: ih.ops.rope(desc, 1 << 20, (1 << 20) + 4 * at))
            seen += 1
    assert seen > 2 * seq * heads


def test_outputs_that_overlap_other_arguments_are_refused():
    M = 1 << 20
    # y: a part of x, of w, of a residual at another place, of the bias and of the gate
    d = linear_desc(m=64, n=8, k=16, dtype="f32", gate_rows=2)
    for x, w, kw in ((M - 4 * 63 * 16, 2 * M, {}), (2 * M, M + 64 * 8 * 4 - 4, {}), (2 * M, 3 * M, dict(d_residual=M + 32)),
                     (2 * M, 3 * M, dict(d_bias=M + 4 * 40)), (2 * M, 3 * M, dict(d_gate=M - 4 * 31 * 8))):
        gate = kw.get("d_gate", 5 * M)
        refused("InvalidArg", "y overlaps", lambda: ih.ops.linear(d, x, w, M, **dict(kw, d_gate=gate)))
    # columns of one buffer, one too far
    d = linear_desc(m=9, n=8, k=16, ldx=24, ldy=24)
    refused("InvalidArg", "y overlaps", lambda: ih.ops.linear(d, M, 2 * M, M + 2 * 15))
    refused("InvalidArg", "y overlaps", lambda: ih.ops.linear(d, M, 2 * M, M - 2 * 7))
    # out over each input, and the workspace over each and over out
    d = cross_desc(batch=2, seq_q=1, seq_kv=100000, dtype="f32")
    need = ih.ops.cross_attention_workspace(d)
    place = dict(d_q=1 * M, d_k=1024 * M, d_v=2048 * M, d_out=3 * M, d_mask=4 * M, d_q_len=5 * M, d_kv_len=6 * M, d_workspace=7 * M)
    for name in ("d_q", "d_k", "d_v", "d_mask", "d_q_len", "d_kv_len", "d_workspace"):
        refused("InvalidArg", "overlaps", lambda: ih.ops.cross_attention(d, **dict(place, d_out=place[name] + 4), workspace_bytes=need))
    for name in ("d_q", "d_k", "d_v", "d_mask", "d_q_len", "d_kv_len", "d_out"):
        refused("InvalidArg", "overlaps", lambda: ih.ops.cross_attention(d, **dict(place, d_workspace=place[name] - 16), workspace_bytes=need))
    d = rope_desc()
    refused("InvalidArg", "overlaps", lambda: ih.ops.rope(d, M, 2 * M, 3 * M, 4 * M, d_positions=2 * M + 64))
    refused("InvalidArg", "overlaps", lambda: ih.ops.rope(d, M, 2 * M, 3 * M, 4 * M, d_lengths=4 * M + 64))
    refused("InvalidArg", "overlaps", lambda: ih.ops.rope(d, M, 2 * M, 3 * M, 2 * M + 64))


def test_numbers_that_the_fields_cannot_hold_are_refused():
    # Their low bits alone would be another, valid call.
    for text, make in (("m of", lambda: linear_desc(m=2 ** 32 + 4)), ("k of", lambda: linear_desc(k=-2 ** 32 + 16)),
                       ("gate_rows of", lambda: linear_desc(gate_rows=2 ** 32)), ("ldx of", lambda: linear_desc(ldx=2 ** 64 + 16)),
                       ("seq_kv of", lambda: cross_desc(seq_kv=2 ** 32 + 7)), ("heads of", lambda: cross_desc(heads=2 ** 33 + 4)),
                       ("mask_stride of", lambda: cross_desc(mask_stride=2 ** 63)), ("stride of", lambda: cross_desc(k_strides=(2 ** 64, 128, 64))),
                       ("first_pos of", lambda: rope_desc(first_pos=2 ** 31)), ("seq of", lambda: rope_desc(seq=2 ** 32 + 5)),
                       ("stride of", lambda: rope_desc(q_strides=(640, 2 ** 63, 64)))):
        refused("Shape", text, make)
    assert rope_desc(first_pos=-2 ** 31).first_pos == -2 ** 31
    for call in (lambda n: ih.ops.linear(linear_desc(), P, 2 * P, 3 * P, d_workspace=4 * P, workspace_bytes=n),
                 lambda n: ih.ops.cross_attention(cross_desc(batch=1, seq_q=1, seq_kv=100000), P, 2 * P, 3 * P, 4 * P, d_workspace=5 * P,
                                                  workspace_bytes=n)):
        refused("InvalidArg", "negative", lambda: call(-1))
