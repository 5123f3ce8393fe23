"""The described operators (rotary positions, linear layer, cross attention) on the GPU against
float64 formulas of the same rounded inputs, one by one and as the half block they make up.

Tolerances are bounds of each element's error, from the arithmetic: u = eps / 2 of the output's
type for its rounding, 2^-24 for each f32 step.
"""
import math

import pytest
import torch

import irodori_hip as ih

pytestmark = pytest.mark.gpu

TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DTYPES = ["bf16", "f16", "f32"]
F = 2.0 ** -24
CANARY = 77.0


def u(dtype):
    return torch.finfo(TYPE[dtype]).eps / 2


def tiny(dtype):
    return torch.finfo(TYPE[dtype]).smallest_normal * u(dtype)


def randn(seed, *shape, dtype="f32", std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(TYPE[dtype]).cuda()


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def close(got, ref, tol, what=""):
    got = got.double()
    err = (got - ref).abs()
    bad = ~(err <= tol)  # a NaN is bad
    if bad.any():
        i = int((err / tol).nan_to_num(nan=math.inf).flatten().argmax())
        raise AssertionError("%s: %d of %d off, worst at %d: got %r want %r tol %r" % (
            what, int(bad.sum()), bad.numel(), i, got.flatten()[i].item(), ref.flatten()[i].item(), tol.flatten()[i].item()))


# ---- rotary positions -----------------------------------------------------------------------
def rope_freq(rot, theta=10000.0, scaling="none", factor=1.0, trained=0.0, fast=32.0, slow=1.0):
    out = []
    for p in range(rot // 2):
        f = (theta * factor ** (rot / (rot - 2)) if scaling == "ntk" else theta) ** (-2 * p / rot)
        if scaling == "linear":
            f /= factor
        if scaling == "by_parts":
            keep = min(1.0, max(0.0, (trained * f / math.tau - slow) / (fast - slow)))
            f *= keep + (1 - keep) / factor
        out.append(f)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def rope_ref(x, pos, freq, layout, rot_heads, amplitude=1.0, inverse=False):
    """The rotated x in float64 and, per element, the sum of its pair's magnitudes."""
    rot = 2 * freq.numel()
    y, mag = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    a = pos.double()[..., None, None] * freq
    c, s = a.cos() * amplitude, a.sin() * amplitude * (-1 if inverse else 1)
    i0 = torch.arange(0, rot, 2, device="cuda") if layout == "interleaved" else torch.arange(rot // 2, device="cuda")
    i1 = i0 + 1 if layout == "interleaved" else i0 + rot // 2
    h = y[:, :, :rot_heads]
    p, q = h[..., i0].clone(), h[..., i1].clone()
    h[..., i0], h[..., i1] = p * c - q * s, p * s + q * c
    mag[:, :, :rot_heads, :, ][..., i0] = (p.abs() + q.abs()) * abs(amplitude)
    mag[:, :, :rot_heads][..., i1] = (p.abs() + q.abs()) * abs(amplitude)
    return y, mag


def rope_tol(ref, mag, dtype):
    # Reduced angle: an f32 of up to pi (2 pi F off), sine and cosine 4 F, products and sum 3 F.
    return u(dtype) * ref.abs() * (1 + F) + 16 * F * mag + tiny(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("b,s,h,hk,d,rot,rh,kw", [
    (2, 75, 16, 16, 64, 64, 8, dict()),
    (1, 1, 4, 1, 128, 64, 4, dict(scaling="by_parts", factor=8.0, trained_len=4096.0)),
    (3, 33, 5, 2, 80, 40, 5, dict(scaling="linear", factor=4.0)),
    (2, 7, 3, 0, 6, 6, 2, dict(theta=100.0)),
    (1, 257, 1, 1, 16, 16, 1, dict()),
    (2, 19, 2, 1, 10, 2, 2, dict(amplitude=1.5)),
    (1, 40, 2, 2, 256, 256, 2, dict(scaling="ntk", factor=4.0, theta=500000.0)),
    (1, 5, 3, 1, 1024, 512, 3, dict()),
    (1, 3, 300, 7, 64, 32, 300, dict(inverse=True)),
])
def test_rope(dtype, layout, b, s, h, hk, d, rot, rh, kw):
    kw = dict(kw)
    far = kw.get("scaling") == "by_parts"
    qkv = randn(1, b, s, h + 2 * hk, d, dtype=dtype)  # keys and queries are slices of one projection
    q, k = qkv[:, :, :h], qkv[:, :, h:h + hk]
    pos = torch.randint(0, 1 << 20, (b, s), generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda() if far else None
    rhk = min(rh, hk)
    desc = ih.RopeDesc(b, s, d, heads=h, kv_heads=hk, dtype=dtype, layout=layout, rot_dim=rot, rot_heads=rh, rot_kv_heads=rhk,
                       first_pos=-3, q_strides=q.stride()[:3], k_strides=k.stride()[:3], **kw)
    qo = torch.full((b, s, h, d), CANARY, dtype=TYPE[dtype], device="cuda")
    ko = torch.full((b, s, max(hk, 1), d), CANARY, dtype=TYPE[dtype], device="cuda")
    ih.ops.rope(desc, ptr(q), ptr(qo), ptr(k) if hk else 0, ptr(ko) if hk else 0, d_positions=ptr(pos), stream=stream())
    p = pos if far else (torch.arange(s, device="cuda") - 3).expand(b, s)
    freq = rope_freq(rot, kw.get("theta", 10000.0), kw.get("scaling", "none"), kw.get("factor", 1.0), kw.get("trained_len", 0.0))
    for x, y, n in ((q, qo, rh), (k, ko, rhk)):
        if x.shape[2] == 0:
            continue
        ref, mag = rope_ref(x, p, freq, layout, n, kw.get("amplitude", 1.0), kw.get("inverse", False))
        close(y, ref, rope_tol(ref, mag, dtype), "rope")
        assert torch.equal(y[:, :, n:], x[:, :, n:]) and torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_rope_in_place_lengths_and_alignment(dtype, offset):
    b, s, h, d = 3, 21, 4, 64
    flat = randn(3, b * s * h * d + offset, dtype=dtype)
    x = flat[offset:].view(b, s, h, d)
    before = x.clone()
    lens = torch.tensor([21, 0, 8], dtype=torch.int32, device="cuda")
    desc = ih.RopeDesc(b, s, d, heads=h, dtype=dtype, rot_dim=32, rot_heads=2, layout="halves")
    ih.ops.rope(desc, ptr(x), ptr(x), d_lengths=ptr(lens), stream=stream())
    ref, mag = rope_ref(before, torch.arange(s, device="cuda").expand(b, s), rope_freq(32), "halves", 2)
    for row, n in enumerate([21, 0, 8]):
        close(x[row, :n], ref[row, :n], rope_tol(ref[row, :n], mag[row, :n], dtype))
        assert torch.equal(x[row, n:], before[row, n:])


def test_rope_far_positions_hold_f32():
    # 2^31 - 2 times the first frequency is 2^31 - 2 radians: an f32 product would be off by 64.
    pos = torch.tensor([[2 ** 31 - 2, 2 ** 30 + 1, 12345678, -(2 ** 31)]], dtype=torch.int32, device="cuda")
    x = randn(4, 1, 4, 2, 64)
    y = torch.empty_like(x)
    ih.ops.rope(ih.RopeDesc(1, 4, 64, heads=2, dtype="f32"), ptr(x), ptr(y), d_positions=ptr(pos), stream=stream())
    ref, mag = rope_ref(x, pos, rope_freq(64), "interleaved", 2)
    # float64 angles of 2^31 radians are off by 2^31 2^-53 on either side, far below F.
    close(y, ref, rope_tol(ref, mag, "f32"))


def test_rope_gradient_is_the_inverse_flag():
    # <rope(x), g> = <x, rope_inverse(g)>, and against differences of the linear map.
    x, g = randn(5, 2, 9, 3, 48), randn(6, 2, 9, 3, 48)
    kw = dict(heads=3, dtype="f32", rot_dim=32, rot_heads=2, layout="halves", amplitude=1.25, scaling="linear", factor=3.0)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    ih.ops.rope(ih.RopeDesc(2, 9, 48, **kw), ptr(x), ptr(y), stream=stream())
    ih.ops.rope(ih.RopeDesc(2, 9, 48, inverse=True, **kw), ptr(g), ptr(dx), stream=stream())
    lhs, rhs = (y.double() * g.double()).sum(), (x.double() * dx.double()).sum()
    assert abs(lhs - rhs) <= 64 * F * (x.double().norm() * g.double().norm())
    e = torch.zeros_like(x)
    e[1, 4, 1, 3] = 0.5
    y2 = torch.empty_like(x)
    ih.ops.rope(ih.RopeDesc(2, 9, 48, **kw), ptr(x + e), ptr(y2), stream=stream())
    diff = ((y2.double() - y.double()) * g.double()).sum() / 0.5
    assert abs(diff - dx[1, 4, 1, 3].double()) <= 64 * F * 8 * g.abs().max().double() * x.abs().max().double()


def test_rope_lengths_below_zero():
    # Lengths of any sign, the lowest number among them: rows without a token stay as they were, the rows beside them too.
    b, s, h, d = 5, 2051, 3, 64
    lens = [-1, -2 ** 31, 2051, 1 - 2 ** 31, 2 ** 31 - 1]
    x = randn(3, b, s, h, d)
    flat = torch.full((b * s * h * d + 4096,), CANARY, device="cuda")
    y = flat[:b * s * h * d].view(b, s, h, d)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ih.ops.rope(ih.RopeDesc(b, s, d, heads=h, dtype="f32"), ptr(x), ptr(y), d_lengths=ptr(n), stream=stream())
    ref, mag = rope_ref(x, torch.arange(s, device="cuda").expand(b, s), rope_freq(64), "interleaved", h)
    for row in range(b):
        if lens[row] < 0:
            assert (y[row] == CANARY).all()
        else:
            close(y[row], ref[row], rope_tol(ref[row], mag[row], "f32"))
    assert (flat[b * s * h * d:] == CANARY).all()


@pytest.mark.parametrize("theta,kw", [(10000.0, dict()), (1.5, dict()), (1.5, dict(scaling="ntk", factor=2.0))])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_rope_far_positions_of_many_pairs(theta, kw, layout):
    # 2^28 times a frequency of half a radian: the frequencies of all 256 pairs have to hold float64 (2^28 2^-53 is F / 2).
    pos = torch.tensor([[2 ** 28 - 1, 2 ** 27 + 1, 12345678, -(2 ** 28)]], dtype=torch.int32, device="cuda")
    x = randn(4, 1, 4, 2, 512)
    y = torch.empty_like(x)
    ih.ops.rope(ih.RopeDesc(1, 4, 512, heads=2, dtype="f32", theta=theta, layout=layout, **kw), ptr(x), ptr(y), d_positions=ptr(pos),
                stream=stream())
    ref, mag = rope_ref(x, pos, rope_freq(512, theta, **kw), layout, 2)
    close(y, ref, rope_tol(ref, mag, "f32"))


def test_rope_between_heads_of_one_buffer():
    # From some heads of a buffer into others, and in place beside them: no element is shared.
    b, s, h, d = 2, 5, 2, 64
    for at in (0, 2, 4):
        buf = randn(1, b, s, 6, d)
        before = buf.clone()
        q, out = buf[:, :, 2:4], buf[:, :, at:at + h]
        desc = ih.RopeDesc(b, s, d, heads=h, dtype="f32", q_strides=q.stride()[:3], q_out_strides=out.stride()[:3])
        ih.ops.rope(desc, ptr(q), ptr(out), stream=stream())
        ref, mag = rope_ref(before[:, :, 2:4], torch.arange(s, device="cuda").expand(b, s), rope_freq(d), "interleaved", h)
        close(out, ref, rope_tol(ref, mag, "f32"))
        rest = [i for i in range(6) if not at <= i < at + h]
        assert torch.equal(buf[:, :, rest], before[:, :, rest])


# ---- linear layer -----------------------------------------------------------------------------
ACTS = {
    "none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
    "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
}


def run_linear(x, w, y, dtype, out, act="none", bias=None, gate=None, gate_rows=0, residual=None, m=None, n=None, k=None):
    m, k = m or x.shape[0], k or x.shape[1]
    n = n or w.shape[0]
    desc = ih.LinearDesc(m, n, k, dtype=dtype, out_dtype=out, activation=act, gate_rows=gate_rows, ldx=x.stride(0), ldw=w.stride(0),
                         ldy=y.stride(0), ldr=residual.stride(0) if residual is not None else None)
    nbytes = ih.ops.linear_workspace(desc)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
    ih.ops.linear(desc, ptr(x), ptr(w), ptr(y), d_bias=ptr(bias), d_gate=ptr(gate), d_residual=ptr(residual), d_workspace=ptr(ws),
                  workspace_bytes=nbytes, stream=stream())


def linear_ref(x, w, out, act="none", bias=None, gate=None, gate_rows=0, residual=None):
    """Float64 result and its tolerance: a sum of k products loses at most k F of their magnitudes; no
    activation here is steeper than 1.13; its own error is a few F of the argument and of 1."""
    m, k = x.shape
    z = x.double() @ w.double().T
    mag = x.double().abs() @ w.double().abs().T
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    y = ACTS[act](z)
    tol = 1.13 * (k + 4) * F * mag + (16 * F * (z.abs() + 1) if act != "none" else 0)
    if gate is not None:
        g = gate.double()[torch.arange(m, device="cuda") // gate_rows]
        y, tol = y * g, (tol + F * y.abs()) * g.abs()
    if residual is not None:
        y = y + residual.double()
        tol = tol + F * y.abs()
    return y, tol + u(out) * (y.abs() + tol) + tiny(out)


SHAPES = [(1, 1, 1), (1, 1024, 512), (2, 96, 2816), (3, 5, 7), (4, 3680, 1280), (15, 64, 250), (16, 100, 64), (17, 33, 65), (32, 64, 64),
          (64, 128, 1000), (65, 1280, 192), (101, 333, 1001), (253, 1280, 1280), (300, 520, 96), (1500, 1024, 128), (1100, 2050, 72),
          (40, 70, 130), (700, 1500, 250), (2100, 4000, 66), (5000, 5632, 64), (6100, 5632, 1024), (12100, 5500, 1032), (1900, 1300, 135)]


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(dtype, out, m, n, k):
    x, w = randn(1, m, k, dtype=dtype), randn(2, n, k, dtype=dtype, std=k ** -0.5)
    bias, res = randn(3, n), randn(4, m, n, dtype=out)
    gate = randn(5, -(-m // 7), n)
    y = torch.full((m, n), CANARY, dtype=TYPE[out], device="cuda")
    run_linear(x, w, y, dtype, out)
    close(y, *linear_ref(x, w, out), "plain")
    run_linear(x, w, y, dtype, out, "silu", bias=bias, gate=gate, gate_rows=7, residual=res)
    close(y, *linear_ref(x, w, out, "silu", bias, gate, 7, res), "all")
    # onto the residual
    ref = linear_ref(x, w, out, "none", bias, None, 0, res)
    run_linear(x, w, res, dtype, out, bias=bias, residual=res)
    close(res, *ref, "in place")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m", [2, 70])
def test_linear_activations(act, m):
    x, w = randn(1, m, 64, std=3.0), randn(2, 40, 64, std=0.3)
    y = torch.empty(m, 40, device="cuda")
    run_linear(x, w, y, "f32", "f32", act)
    close(y, *linear_ref(x, w, "f32", act), act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 65, 40), (5, 24, 333), (40, 70, 129), (130, 260, 128)])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (3, 1), (2, 2)])
def test_linear_strides_and_alignment(dtype, m, n, k, pad, offset):
    """Rows apart and off every wide boundary; what lies between and around them is neither read into
    the result (NaN there) nor written."""
    def rows(seed, r, c, dt):
        flat = torch.full(((r + 1) * (c + pad) + offset + 64,), math.nan, dtype=TYPE[dt], device="cuda")
        v = flat[offset:offset + r * (c + pad)].view(r, c + pad)[:, :c]
        v.copy_(randn(seed, r, c, dtype=dt))
        return flat, v
    _, x = rows(1, m, k, dtype)
    _, w = rows(2, n, k, dtype)
    flat, y = rows(3, m, n, dtype)
    flat.fill_(CANARY)
    run_linear(x, w, y, dtype, dtype)
    close(y, *linear_ref(x, w, dtype), "strided")
    kept = torch.ones_like(flat, dtype=torch.bool)
    kept[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n] = False
    assert (flat[kept] == CANARY).all()


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("m,n,k,pad", [(1003, 1283, 1288, 8), (403, 2819, 2824, 8), (1501, 1291, 128, 8), (2101, 2051, 72, 8),
                                       (1501, 5635, 3688, 8), (1902, 1801, 136, 3), (901, 1030, 136, 3)])
def test_linear_edges_of_large_tiles(dtype, out, m, n, k, pad):
    """Tiles of every size that end past the last row and inside a lane's columns, everything after the product
    with them, onto the residual; the columns between rows keep what they hold."""
    def rows(seed, r, c, dt):
        flat = torch.full((r, c + pad), math.nan, dtype=TYPE[dt], device="cuda")
        v = flat[:, :c]
        v.copy_(randn(seed, r, c, dtype=dt))
        return flat, v
    _, x = rows(1, m, k, dtype)
    _, w = rows(2, n, k, dtype)
    w.mul_(k ** -0.5)
    bias, gate = randn(3, n), randn(5, -(-m // 7), n)
    flat, y = rows(4, m, n, out)
    flat[:, n:] = CANARY
    ref = linear_ref(x, w, out, "silu", bias, gate, 7, y.clone())
    run_linear(x, w, y, dtype, out, "silu", bias=bias, gate=gate, gate_rows=7, residual=y)
    close(y, *ref, "edges")
    assert (flat[:, n:] == CANARY).all()


def test_linear_broadcast_rows_and_specials():
    # A stride of 0 repeats one row of x and of the residual; infinities and NaN reach their own rows only.
    w = randn(2, 48, 64, dtype="bf16")
    x, res = randn(1, 1, 64, dtype="bf16"), randn(3, 1, 48, dtype="bf16")
    y = torch.empty(5, 48, dtype=torch.bfloat16, device="cuda")
    run_linear(x.expand(5, 64), w, y, "bf16", "bf16", residual=res.expand(5, 48))
    ref, tol = linear_ref(x.expand(5, 64), w, "bf16", residual=res.expand(5, 48))
    close(y, ref, tol)
    x = randn(4, 70, 64, dtype="bf16")
    x[3, 5], x[40, 0] = math.nan, math.inf
    y = torch.empty(70, 48, dtype=torch.bfloat16, device="cuda")
    run_linear(x, w, y, "bf16", "bf16", "relu")
    assert y[3].isnan().all() and ((y[40] == math.inf) | (y[40] == 0)).all()
    rest = [i for i in range(70) if i not in (3, 40)]
    ref, tol = linear_ref(x[rest], w, "bf16", "relu")
    close(y[rest], ref, tol)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("m", [16, 300])
def test_linear_tanh_of_small_arguments(dtype, out, m):
    """Relative to the result, however small: the argument is one exact product."""
    n = 64
    z = torch.logspace(-30, 1.2, m, dtype=torch.float64).to(TYPE[dtype]).cuda()
    z[::2] *= -1
    w = torch.ones(n, 1, dtype=TYPE[dtype], device="cuda")
    y = torch.empty(m, n, dtype=TYPE[out], device="cuda")
    run_linear(z[:, None].contiguous(), w, y, dtype, out, "tanh")
    ref = torch.tanh(z.double())[:, None].expand(m, n)
    # z + z^3 P(z^2) is off by 2 F (6 with one coefficient).  1 - t: t has an exponential of a rounded argument, a sum and a
    # reciprocal, 6 F of it, and there is less of it than 1.2 of the result from 1/2 on (15 from 1/16 on); then a rounding.
    close(y, ref, ((10 if out == "f32" else 90) * F + u(out)) * ref.abs() + tiny(out), "tanh")


@pytest.mark.parametrize("m", [9, 200])
def test_linear_between_columns_of_one_buffer(m):
    # x, y and the residual are columns of one buffer; w stands before it.
    k, n = 64, 48
    buf = randn(1, m, k + 2 * n)
    before, w = buf.clone(), randn(2, n, k, std=k ** -0.5)
    x, res, y = buf[:, n:n + k], buf[:, n + k:], buf[:, :n]
    ref = linear_ref(x, w, "f32", "none", None, None, 0, res.clone())
    run_linear(x, w, y, "f32", "f32", residual=res)
    close(y, *ref, "columns")
    assert torch.equal(buf[:, n:], before[:, n:])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m", [5, 40, 700])
def test_linear_rows_far_apart(dtype, m):
    # Rows 2^22 bytes and more apart, past the windows of the asynchronous loads; 700 of x past 2^32 bytes.
    n, k = 40, 70
    step = (1 << 23) // TYPE[dtype].itemsize
    x = torch.empty((m - 1) * step + k, dtype=TYPE[dtype], device="cuda").as_strided((m, k), (step, 1))
    w = torch.empty((n - 1) * step + k, dtype=TYPE[dtype], device="cuda").as_strided((n, k), (step, 1))
    x.copy_(randn(1, m, k, dtype=dtype)), w.copy_(randn(2, n, k, dtype=dtype, std=k ** -0.5))
    y = torch.empty(m, n, dtype=TYPE[dtype], device="cuda")
    run_linear(x, w, y, dtype, dtype)
    close(y, *linear_ref(x, w, dtype), "far apart")


@pytest.mark.parametrize("dtype,k", [("bf16", (1 << 21) + 3), ("f32", (1 << 20) + 3)])
@pytest.mark.parametrize("m", [3, 18])
def test_linear_long_reduction(dtype, k, m):
    x, w = randn(1, m, k, dtype=dtype), randn(2, 33, k, dtype=dtype, std=k ** -0.5)
    y = torch.empty(m, 33, device="cuda")
    run_linear(x, w, y, dtype, "f32")
    close(y, *linear_ref(x, w, "f32"), "long")


# ---- cross attention --------------------------------------------------------------------------
def run_cross(q, k, v, out, dtype, mask=None, q_len=None, kv_len=None, scale=None):
    b, sq, h, d = q.shape
    skv, hk = k.shape[1], k.shape[2]
    desc = ih.CrossAttentionDesc(b, sq, skv, h, hk, d, dtype=dtype, scale=scale, q_strides=q.stride()[:3], k_strides=k.stride()[:3],
                                 v_strides=v.stride()[:3], out_strides=out.stride()[:3],
                                 mask_stride=mask.stride(0) if mask is not None else None)
    nbytes = ih.ops.cross_attention_workspace(desc)
    ws = torch.full((max(nbytes, 1),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN: nothing of it may be read before it is written
    ih.ops.cross_attention(desc, ptr(q), ptr(k), ptr(v), ptr(out), d_mask=ptr(mask), d_q_len=ptr(q_len), d_kv_len=ptr(kv_len),
                           d_workspace=ptr(ws), workspace_bytes=nbytes, stream=stream())


def check_cross(got, q, k, v, dtype, mask=None, q_len=None, kv_len=None, scale=None, what="cross"):
    """Against float64, row by row: scores lose (d + 4) F of their magnitudes (twice: the row's
    largest too), exp2 and the sums 2^-20 with them, p and the result u each in the 16-bit forms."""
    b, sq, h, d = q.shape
    skv, hk = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    for i in range(b):
        n = skv if kv_len is None else max(0, min(skv, int(kv_len[i])))
        keys = torch.arange(n, device="cuda")
        if mask is not None:
            keys = keys[mask[i, :n] != 0]
        toks = sq if q_len is None else max(0, min(sq, int(q_len[i])))
        if keys.numel() == 0:
            assert (got[i, :toks] == 0).all(), what
            continue
        qi = q[i, :toks].double().transpose(0, 1)  # [h, toks, d]
        ki = k[i, keys].double().transpose(0, 1).repeat_interleave(h // hk, 0)
        vi = v[i, keys].double().transpose(0, 1).repeat_interleave(h // hk, 0)
        s = torch.matmul(qi, ki.transpose(1, 2).contiguous()) * scale
        p = torch.softmax(s, dim=-1)
        ref = torch.matmul(p, vi)
        mag = torch.matmul(p, vi.abs())
        smag = (torch.matmul(qi.abs(), ki.abs().transpose(1, 2).contiguous()) * abs(scale)).amax(-1, keepdim=True)
        rel = 2 * (d + 4) * F * smag + 2.0 ** -20 + (u(dtype) if dtype != "f32" else skv * F)
        tol = rel * mag + u(dtype) * ref.abs() * (1 + 2.0 ** -6) + tiny(dtype)
        if dtype == "f16":  # probabilities below the smallest normal are off by 2^-25 at most
            tol = tol + 2.0 ** -25 * vi.abs().sum(1, keepdim=True)
        close(got[i, :toks].transpose(0, 1), ref, tol, "%s row %d" % (what, i))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,sq,skv,h,hk", [(1, 1, 1, 1, 1), (2, 1, 63, 4, 2), (1, 33, 64, 2, 2), (3, 7, 65, 6, 2), (2, 101, 37, 3, 3),
                                           (1, 130, 200, 4, 1), (2, 1, 700, 8, 2), (1, 64, 4200, 2, 1), (2, 300, 129, 2, 2)])
def test_cross_attention(dtype, d, b, sq, skv, h, hk):
    q, kv = randn(1, b, sq, h, d, dtype=dtype), randn(2, b, skv, 2, hk, d, dtype=dtype)
    k, v = kv[:, :, 0], kv[:, :, 1]
    out = torch.full((b, sq, h, d), CANARY, dtype=TYPE[dtype], device="cuda")
    run_cross(q, k, v, out, dtype)
    check_cross(out, q, k, v, dtype)
    mask = (torch.rand(b, skv, generator=torch.Generator().manual_seed(3)) < 0.6).to(torch.uint8).cuda() * 255
    mask[-1] = 0
    run_cross(q, k, v, out, dtype, mask=mask)
    check_cross(out, q, k, v, dtype, mask=mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 5, 70])
def test_cross_attention_lengths_masks_and_what_they_hide(dtype, sq):
    """Lengths of every kind, keys and values that are NaN or infinite wherever they do not count,
    queries that are NaN past their length, outputs past it untouched."""
    b, skv, h, hk, d = 8, 333, 4, 2, 64
    lens = torch.tensor([333, 0, 1, 64, 65, 200, -5, 10000], dtype=torch.int32, device="cuda")
    q_len = torch.tensor([sq, sq, max(1, sq - 1), 1, 0, sq, sq, 10000], dtype=torch.int32, device="cuda")
    mask = (torch.rand(b, skv + 5, generator=torch.Generator().manual_seed(3)) < 0.7).to(torch.uint8).cuda()[:, :skv]
    mask[5, :128] = 0  # whole tiles
    mask[0, 64:128] = 0
    mask[2, 0] = 1
    q, k, v = randn(1, b, sq, h, d, dtype=dtype), randn(2, b, skv, hk, d, dtype=dtype), randn(4, b, skv, hk, d, dtype=dtype)
    for i in range(b):
        n = max(0, min(skv, int(lens[i])))
        off = torch.ones(skv, dtype=torch.bool, device="cuda")
        off[:n] = mask[i, :n] == 0
        k[i, off], v[i, off] = math.nan, math.inf
        v[i, off.nonzero()[::2, 0]] = math.nan
        q[i, max(0, min(sq, int(q_len[i]))):] = math.nan
    out = torch.full((b, sq, h, d), CANARY, dtype=TYPE[dtype], device="cuda")
    run_cross(q, k, v, out, dtype, mask=mask, q_len=q_len, kv_len=lens)
    check_cross(out, q, k, v, dtype, mask=mask, q_len=q_len, kv_len=lens)
    for i in range(b):
        assert (out[i, max(0, min(sq, int(q_len[i]))):] == CANARY).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [130], [0, 3, 0], [5000, 1, 0, 700, 64], [0] * 70 + [200] + [0] * 9 + [4999, 1], [65] * 90])
def test_cross_attention_split_over_short_rows(dtype, d, lens):
    """A description of many keys, split, of which the rows hold few: runs that are empty, that end
    inside a row and that span several; more rows than a wavefront has lanes."""
    b, sq, skv, h, hk = len(lens), 2, 5000, 4, 2
    desc = ih.CrossAttentionDesc(b, sq, skv, h, hk, d, dtype=dtype)
    assert ih.ops.cross_attention_workspace(desc) > 0
    q = randn(1, b, sq, h, d, dtype=dtype)
    k, v = (randn(i, 1, skv, hk, d, dtype=dtype).expand(b, skv, hk, d) for i in (2, 3))  # (one set of states)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    mask = (torch.rand(b, skv, generator=torch.Generator().manual_seed(3)) < 0.5).to(torch.uint8).cuda()
    q_len = torch.tensor([i % 3 for i in range(b)], dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(mask=mask, q_len=q_len)):
        out = torch.full((b, sq, h, d), CANARY, dtype=TYPE[dtype], device="cuda")
        run_cross(q, k, v, out, dtype, kv_len=n, **kw)
        check_cross(out, q, k, v, dtype, kv_len=n, **kw)
        for i in range(b):
            assert (out[i, int(q_len[i]) if kw else sq:] == CANARY).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pad,offset", [(2, 0), (1, 1), (3, 0)])
def test_cross_attention_strides_and_alignment(dtype, d, pad, offset):
    b, sq, skv, h, hk = 2, 40, 150, 4, 2

    def tensor(seed, s, n):
        flat = torch.full((b * s * n * (d + pad) + offset + 64,), math.nan, dtype=TYPE[dtype], device="cuda")
        t = flat[offset:offset + b * s * n * (d + pad)].view(b, s, n, d + pad)[..., :d]
        t.copy_(randn(seed, b, s, n, d, dtype=dtype))
        return flat, t
    (_, q), (_, k), (_, v), (flat, out) = tensor(1, sq, h), tensor(2, skv, hk), tensor(3, skv, hk), tensor(4, sq, h)
    flat.fill_(CANARY)
    run_cross(q, k, v, out, dtype)
    check_cross(out, q, k, v, dtype)
    kept = torch.ones_like(flat, dtype=torch.bool)
    kept[offset:offset + b * sq * h * (d + pad)].view(b, sq, h, d + pad)[..., :d] = False
    assert (flat[kept] == CANARY).all()
    # head-major operands and output
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    ot = torch.empty(b, h, sq, d, dtype=TYPE[dtype], device="cuda").transpose(1, 2)
    run_cross(qt, kt, vt, ot, dtype)
    assert torch.equal(ot, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,skv", [(1, 9000), (40, 600)])
def test_cross_attention_scores_that_grow(dtype, sq, skv):
    """Scores that rise over the keys move the softmax reference at almost every tile; and scores of
    +-60 000 in one row."""
    b, h, hk, d = 1, 2, 1, 64
    q = torch.ones(b, sq, h, d, dtype=TYPE[dtype], device="cuda")
    q[:, :, 1] = -1
    ramp = (torch.arange(skv, device="cuda") * (512 / skv)).floor() / 8  # exact in every type
    k = ramp.to(TYPE[dtype])[None, :, None, None].expand(b, skv, hk, d).contiguous()
    v = randn(3, b, skv, hk, d, dtype=dtype)
    out = torch.empty(b, sq, h, d, dtype=TYPE[dtype], device="cuda")
    run_cross(q, k, v, out, dtype, scale=0.5)
    check_cross(out, q, k, v, dtype, scale=0.5)
    for scale in (0.0, -0.5, 2.0 ** -10, 15.0, 1e-42):
        run_cross(q, k, v, out, dtype, scale=scale)
        check_cross(out, q, k, v, dtype, scale=scale, what="scale %g" % scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_attention_infinite_scores(dtype):
    # Keys of -inf score nothing while another key is there; a row of nothing else gives 0; +inf and NaN give NaN.
    q = torch.ones(1, 3, 1, 64, dtype=TYPE[dtype], device="cuda")
    k, v = randn(2, 1, 200, 1, 64, dtype=dtype), randn(3, 1, 200, 1, 64, dtype=dtype)
    k[:, :100] = -math.inf
    out = torch.empty_like(q)
    run_cross(q, k, v, out, dtype)
    check_cross(out, q, k[:, 100:], v[:, 100:], dtype)
    k[:] = -math.inf
    run_cross(q, k, v, out, dtype)
    assert (out == 0).all()
    for bad in (math.inf, math.nan):
        k[:] = 0
        k[0, 150, 0, 7] = bad
        run_cross(q, k, v, out, dtype)
        assert out.isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cross_attention_offsets_past_32_bits(dtype):
    # Keys 2^20 elements apart: the last of 2300 lies past 2^31 elements (and 2^32 bytes).
    skv, step = 2300, 1 << 20
    flat = torch.empty(skv * step, dtype=TYPE[dtype], device="cuda")
    kv = flat.view(1, skv, step)[:, :, :128].view(1, skv, 2, 64)
    kv.copy_(randn(1, 1, skv, 2, 64, dtype=dtype))
    k, v = kv[:, :, :1], kv[:, :, 1:]
    for sq in (1, 66):
        q, out = randn(2, 1, sq, 2, 64, dtype=dtype), torch.empty(1, sq, 2, 64, dtype=TYPE[dtype], device="cuda")
        run_cross(q, k, v, out, dtype)
        check_cross(out, q, k, v, dtype)


def test_cross_attention_broadcast_keys():
    # One set of states for every batch row (stride 0), and one head for all.
    q = randn(1, 3, 20, 4, 64, dtype="bf16")
    k, v = randn(2, 1, 90, 1, 64, dtype="bf16").expand(3, 90, 1, 64), randn(3, 1, 90, 1, 64, dtype="bf16").expand(3, 90, 1, 64)
    out = torch.empty_like(q)
    run_cross(q, k, v, out, "bf16")
    check_cross(out, q, k, v, "bf16")
    wide = torch.empty_like(q)
    run_cross(q, k.expand(3, 90, 4, 64), v.expand(3, 90, 4, 64), wide, "bf16")
    check_cross(wide, q, k, v, "bf16")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,sq,skv", [(64, 5, 37), (64, 300, 70), (128, 40, 33), (64, 1, 3001)])
def test_cross_attention_one_value_for_all_keys(dtype, d, sq, skv):
    # A token stride of 0: every key's value is the same row, and so is the result, infinities included.
    q, k = randn(1, 2, sq, 2, d, dtype=dtype), randn(2, 2, skv, 2, d, dtype=dtype)
    row = randn(3, 2, 1, 2, d, dtype=dtype)
    row[0, 0, 1, 3], row[1, 0, 0, 9] = float("inf"), float("-inf")
    out = torch.empty_like(q)
    run_cross(q, k, row.expand(2, skv, 2, d), out, dtype)
    want = row.expand(2, sq, 2, d)
    finite = want.isfinite()
    assert torch.equal(out[~finite], want[~finite])
    # The weights' sum is off by its own roundings alone: those of skv f32 additions on both sides.
    tol = (2 * skv * F + 2.0 ** -20 + u(dtype) * (1 + 2.0 ** -6)) * want.double().abs() + tiny(dtype)
    close(out[finite], want.double()[finite], tol[finite], "one value")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cross_attention_strides_of_single_dimensions(dtype):
    # One key, one token, one head or one batch row: that dimension's stride may be anything.
    q, k, v = (randn(i, 1, 1, 1, 64, dtype=dtype) for i in (1, 2, 3))
    for odd in (-1, 1, 2 ** 62):
        desc = ih.CrossAttentionDesc(1, 1, 1, 1, 1, 64, dtype=dtype, q_strides=(odd,) * 3, k_strides=(odd,) * 3, v_strides=(odd,) * 3,
                                     out_strides=(odd,) * 3)
        out = torch.empty_like(q)
        ih.ops.cross_attention(desc, ptr(q), ptr(k), ptr(v), ptr(out), stream=stream())
        assert torch.equal(out, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq", [1, 70])
@pytest.mark.parametrize("masked", [False, True])
def test_cross_attention_single_key(dtype, d, sq, masked):
    """One key: its weight is 1, and the result its value, infinities and NaN among them."""
    b, h = 3, 2
    q, k, v = randn(1, b, sq, h, d, dtype=dtype), randn(2, b, 1, h, d, dtype=dtype), randn(3, b, 1, h, d, dtype=dtype)
    for i, x in enumerate((math.inf, -math.inf, math.nan)):
        v[:, 0, 1, 7 * i] = x
    mask = torch.tensor([[1], [255], [0]], dtype=torch.uint8, device="cuda") if masked else None
    out = torch.full((b, sq, h, d), CANARY, dtype=TYPE[dtype], device="cuda")
    run_cross(q, k, v, out, dtype, mask=mask)
    want = v.expand(b, sq, h, d).clone()
    if masked:
        want[2] = 0
    special = ~want.isfinite()
    assert torch.equal(out[special].nan_to_num(CANARY), want[special].nan_to_num(CANARY))
    # The product with the weight, the reciprocal of the same weight and their product: F each, then the type's rounding.
    close(out[~special], want.double()[~special], (4 * F + u(dtype) * (1 + 4 * F)) * want.double().abs()[~special] + tiny(dtype), "one key")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cross_attention_keys_far_apart(dtype):
    # Keys 2^26 elements apart: inside one tile their byte offsets pass 2^32.
    skv, step = 40, 1 << 26
    flat = torch.empty((skv - 1) * step + 256, dtype=TYPE[dtype], device="cuda")
    kv = flat.as_strided((1, skv, 4, 64), (0, step, 64, 1))
    kv.copy_(randn(1, 1, skv, 4, 64, dtype=dtype))
    k, v = kv[:, :, :2], kv[:, :, 2:]
    for sq in (1, 66):
        q, out = randn(2, 1, sq, 2, 64, dtype=dtype), torch.empty(1, sq, 2, 64, dtype=TYPE[dtype], device="cuda")
        run_cross(q, k, v, out, dtype)
        check_cross(out, q, k, v, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,skv,low", [(1, 9000, 6000), (40, 600, 200), (300, 600, 64), (3, 100, 99)])
def test_cross_attention_first_scores_far_below_the_rest(dtype, sq, skv, low):
    """Keys that a first component puts out of reach come first: the softmax of the others loses nothing by it."""
    big = 60000.0 if dtype == "f16" else 1e15
    q, k, v = (randn(i, 2, n, 2, 64, dtype=dtype) for i, n in ((1, sq), (2, skv), (3, skv)))
    q[..., 0] = big
    k[..., 0] = 0
    k[:, :low, :, 0] = -big
    out = torch.empty_like(q)
    run_cross(q, k, v, out, dtype)
    check_cross(out, q, k[:, low:], v[:, low:], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 1e-42])
def test_cross_attention_scales_next_to_zero(dtype, scale):
    # However large the products, 0 times them is 0, and so is the lowest scale times them nearly.
    big = 60000.0 if dtype == "f16" else 2e18
    q, k, v = (randn(i, 2, n, 2, 64, dtype=dtype) for i, n in ((1, 5), (2, 300), (3, 300)))
    q, k = q.sign() * big, k.sign() * big
    out = torch.empty_like(q)
    mask = (torch.rand(2, 300, generator=torch.Generator().manual_seed(3)) < 0.6).to(torch.uint8).cuda()
    run_cross(q, k, v, out, dtype, mask=mask, scale=scale)
    check_cross(out, q, k, v, dtype, mask=mask, scale=scale)


@pytest.mark.parametrize("d,sq", [(64, 40), (128, 1), (128, 40)])
def test_cross_attention_few_rows_do_not_depend_on_the_batch(d, sq):
    # However many batch rows: 64 rows a workgroup, in two key groups (and not 128, most of which would not exist).
    b, skv, h, dtype = 40, 900, 20, "f32"
    q, k, v = randn(1, b, sq, h, d, dtype=dtype), randn(2, b, skv, h, d, dtype=dtype), randn(3, b, skv, h, d, dtype=dtype)
    out, few = torch.empty_like(q), torch.empty_like(q[:10])
    for n, o in ((b, out), (10, few)):
        assert ih.ops.cross_attention_workspace(ih.CrossAttentionDesc(n, sq, skv, h, h, d, dtype=dtype)) == 0
        run_cross(q[:n], k[:n], v[:n], o, dtype)
    assert torch.equal(out[:10], few)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,h,hk", [(1, 20, 20), (9, 80, 20), (64, 20, 20), (65, 20, 20)])
def test_cross_attention_many_batch_rows(dtype, d, sq, h, hk):
    b, skv = 27, 133
    q, k, v = randn(1, b, sq, h, d, dtype=dtype), randn(2, b, skv, hk, d, dtype=dtype), randn(3, b, skv, hk, d, dtype=dtype)
    lens = torch.tensor([(skv - 17 * i) % (skv + 1) for i in range(b)], dtype=torch.int32, device="cuda")
    mask = (torch.rand(b, skv, generator=torch.Generator().manual_seed(3)) < 0.6).to(torch.uint8).cuda()
    out = torch.full((b, sq, h, d), CANARY, dtype=TYPE[dtype], device="cuda")
    run_cross(q, k, v, out, dtype, mask=mask, kv_len=lens)
    check_cross(out, q, k, v, dtype, mask=mask, kv_len=lens)


def test_cross_attention_into_a_part_of_the_queries_buffer():
    b, sq, skv, h, d = 2, 9, 70, 2, 64
    buf = randn(1, b, sq, 3 * h, d)
    before, k, v = buf.clone(), randn(2, b, skv, h, d), randn(3, b, skv, h, d)
    run_cross(buf[:, :, h:2 * h], k, v, buf[:, :, :h], "f32")
    check_cross(buf[:, :, :h], before[:, :, h:2 * h], k, v, "f32")
    assert torch.equal(buf[:, :, h:], before[:, :, h:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,skv", [(1, 1), (1, 9000), (40, 300), (300, 70)])
@pytest.mark.parametrize("sign", [1, -1])
def test_cross_attention_equal_scores_of_any_size(dtype, d, sq, skv, sign):
    """Every key at one score, up to the type's lowest and largest value: the plain mean of the values."""
    q, k, v = (torch.zeros(1, n, 2, d, dtype=TYPE[dtype], device="cuda") for n in (sq, skv, skv))
    v.copy_(randn(3, 1, skv, 2, d, dtype=dtype))
    want, mag = v.double().mean(1, keepdim=True).expand(1, sq, 2, d), v.double().abs().mean(1, keepdim=True).expand(1, sq, 2, d)
    for big in (1e3, 6e4) + ((1e9, 1.7e15, 3e30, torch.finfo(TYPE[dtype]).max) if dtype != "f16" else (65504.0,)):
        k[..., 0] = sign * big
        q[..., 0] = (1 + torch.rand(sq, 2, generator=torch.Generator().manual_seed(5))).to(TYPE[dtype]).cuda()
        q[..., 1], k[..., 1] = 60000 if dtype == "f16" else 0, sign * big if dtype == "f16" else 0
        out = torch.full_like(q, CANARY)
        run_cross(q, k, v, out, dtype)
        # A product above f32's largest value is an infinite score: NaN, or below all others, with no other there 0.
        inf = (q[..., 0].double() * big > torch.finfo(torch.float32).max * (1 + F / 2))[..., None].expand_as(out)
        assert (out[inf].isnan() if sign > 0 else out[inf] == 0).all()
        # Weights of exactly 1: the sums' roundings, the reciprocal's, the output's.
        tol = (skv + 4) * F * mag + u(dtype) * want.abs() * (1 + 2.0 ** -6) + tiny(dtype)
        close(out[~inf], want[~inf], tol[~inf], "%g" % big)


# ---- the half block they make up ----------------------------------------------------------------
class HalfBlock:
    """x + g * (cross(rope(norm(x) Wq + bq), states Wk, states Wv) Wo), each step one operator."""

    def __init__(self, b, s, t, d, h, hk, ds, dtype):
        self.shape, self.dtype = (b, s, t, d, h, hk, ds), dtype
        dh = d // h
        tt = TYPE[dtype]
        self.norm = 1 + 0.1 * randn(10, d)
        self.wq, self.bq = randn(11, d, d, dtype=dtype, std=d ** -0.5), randn(12, d, std=0.1)
        self.wkv = randn(13, 2 * hk * dh, ds, dtype=dtype, std=ds ** -0.5)
        self.wo, self.gate = randn(14, d, d, dtype=dtype, std=d ** -0.5), randn(15, b, d, std=0.5)
        e = lambda *sh, dt=tt: torch.empty(*sh, dtype=dt, device="cuda")  # noqa: E731
        self.n32, self.n16, self.q, self.kv, self.o = e(b * s, d, dt=torch.float32), e(b * s, d), e(b, s, h, dh), e(b, t, 2, hk, dh), e(b, s, h, dh)
        kw = dict(dtype=dtype)
        self.dq, self.dkv = ih.LinearDesc(b * s, d, d, **kw), ih.LinearDesc(b * t, 2 * hk * dh, ds, **kw)
        self.do = ih.LinearDesc(b * s, d, d, out_dtype="f32", gate_rows=s, **kw)
        self.dr = ih.RopeDesc(b, s, dh, heads=h, layout="halves", scaling="ntk", factor=2.0, **kw)
        self.dk = ih.RopeDesc(b, t, dh, heads=hk, layout="halves", scaling="ntk", factor=2.0, q_strides=self.kv.stride()[0:2] + (dh,),
                              q_out_strides=self.kv.stride()[0:2] + (dh,), **kw)
        self.dx = ih.CrossAttentionDesc(b, s, t, h, hk, dh, k_strides=self.kv.stride()[0:2] + (dh,),
                                        v_strides=self.kv.stride()[0:2] + (dh,), **kw)
        self.nws = max(ih.ops.cross_attention_workspace(self.dx), *(ih.ops.linear_workspace(x) for x in (self.dq, self.dkv, self.do)))
        self.ws = e(max(self.nws, 16), dt=torch.uint8)

    def __call__(self, x, states, kv_len):
        """In place on x [b * s, d] f32."""
        b, s, t, d, h, hk, ds = self.shape
        st, ws = stream(), dict(d_workspace=ptr(self.ws), workspace_bytes=self.nws, stream=stream())
        ih.ops.rms_norm(ptr(x), ptr(self.norm), b * s, d, 1e-5, ptr(self.n32), stream=st)
        n = self.n32
        if self.dtype != "f32":
            self.n16.copy_(self.n32)
            n = self.n16
        ih.ops.linear(self.dq, ptr(n), ptr(self.wq), ptr(self.q), d_bias=ptr(self.bq), **ws)
        ih.ops.linear(self.dkv, ptr(states), ptr(self.wkv), ptr(self.kv), **ws)
        ih.ops.rope(self.dr, ptr(self.q), ptr(self.q), stream=st)
        ih.ops.rope(self.dk, ptr(self.kv), ptr(self.kv), stream=st)
        k, v = self.kv[:, :, 0], self.kv[:, :, 1]
        ih.ops.cross_attention(self.dx, ptr(self.q), ptr(k), ptr(v), ptr(self.o), d_kv_len=ptr(kv_len), **ws)
        ih.ops.linear(self.do, ptr(self.o), ptr(self.wo), ptr(x), d_gate=ptr(self.gate), d_residual=ptr(x), **ws)

    def reference(self, x, states, kv_len):
        b, s, t, d, h, hk, ds = self.shape
        dh = d // h
        x = x.double()
        n = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * self.norm.double()
        q = (n @ self.wq.double().T + self.bq.double()).view(b, s, h, dh)
        kv = (states.double() @ self.wkv.double().T).view(b, t, 2, hk, dh)
        f = rope_freq(dh, scaling="ntk", factor=2.0)
        q, _ = rope_ref(q, torch.arange(s, device="cuda").expand(b, s), f, "halves", h)
        k, _ = rope_ref(kv[:, :, 0], torch.arange(t, device="cuda").expand(b, t), f, "halves", hk)
        sc = torch.einsum("bshd,bthd->bhst", q, k.repeat_interleave(h // hk, 2)) * dh ** -0.5
        sc = sc.masked_fill((torch.arange(t, device="cuda")[None] >= kv_len[:, None])[:, None, None], -math.inf)
        o = torch.einsum("bhst,bthd->bshd", torch.softmax(sc, -1).nan_to_num(0.0), kv[:, :, 1].repeat_interleave(h // hk, 2))
        return x + (o.reshape(b, s, d) @ self.wo.double().T * self.gate.double()[:, None]).reshape(b * s, d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,t,h,hk", [(2, 75, 61, 4, 4), (3, 1, 900, 4, 2)])
def test_half_block(dtype, b, s, t, h, hk):
    d, ds = 256, 192
    blk = HalfBlock(b, s, t, d, h, hk, ds, dtype)
    x, states = randn(20, b * s, d), randn(21, b * t, ds, dtype=dtype)
    kv_len = torch.tensor([t, 0, t // 2][:b], dtype=torch.int32, device="cuda")
    ref = blk.reference(x, states, kv_len)
    y = x.clone()
    blk(y, states, kv_len)
    # Five roundings to the operand type of uncorrelated factors (norm, q, q rotated, k, k rotated, p, v, o) of
    # the increment, each u relative to its own norm; scores of order 1 pass theirs on once.
    inc, want = (y.double() - x.double()), (ref - x.double())
    assert (inc - want).norm() <= (8 * u(dtype) + 2.0 ** -19) * want.norm()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_half_block_captured_and_on_another_stream(dtype):
    """Captured from the first call on a stream of its own, replayed between eager work, against eager
    calls bit for bit; two blocks with a workspace each on two streams at once."""
    b, s, t, d, h, hk, ds = 2, 3, 2100, 256, 4, 2, 192
    states = randn(21, b * t, ds, dtype=dtype)
    kv_len = torch.tensor([t, 700], dtype=torch.int32, device="cuda")
    x0 = randn(20, b * s, d)
    blk = HalfBlock(b, s, t, d, h, hk, ds, dtype)
    x = x0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        blk(x, states, kv_len)
    want = x0.clone()
    other = HalfBlock(b, s, t, d, h, hk, ds, dtype)
    other(want, states, kv_len)
    for i in range(4):
        x.copy_(x0)
        graph.replay()
        y = x0.clone()
        other(y, states, kv_len)
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, want)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    a, c = x0.clone(), x0.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        blk(a, states, kv_len)
    with torch.cuda.stream(s2):
        other(c, states, kv_len)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(c, want)


CHILD = """
import torch
import irodori_hip as ih

def captured(name, call, *outs):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(torch.cuda.current_stream().cuda_stream)
    got = []
    for _ in range(3):
        for o in outs:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        got.append([o.clone() for o in outs])
    for o in outs:
        o.zero_()
    call(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for rep in got:
        for a, o in zip(rep, outs):
            assert o.float().abs().sum() > 0 and torch.equal(a, o), name
    print(name, flush=True)

t = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
for m, n, k in ((3, 64, 64), (40, 64, 64), (600, 512, 128), (12000, 5632, 1024), (40, 64, 33)):
    x, w, y = t(m, k), t(n, k), t(m, n)
    d = ih.LinearDesc(m, n, k)
    captured("linear %d" % m, lambda s: ih.ops.linear(d, x.data_ptr(), w.data_ptr(), y.data_ptr(), stream=s), y)
q, qo = t(2, 9, 4, 64), t(2, 9, 4, 64)
rd = ih.RopeDesc(2, 9, 64, heads=4)
captured("rope", lambda s: ih.ops.rope(rd, q.data_ptr(), qo.data_ptr(), stream=s), qo)
for sq, skv, dim in ((1, 9000, 128), (70, 90, 128), (2000, 90, 128), (1, 9000, 64), (9000, 90, 64)):
    q, o, kv = t(1, sq, 8, dim), t(1, sq, 8, dim), t(1, skv, 8, dim)
    cd = ih.CrossAttentionDesc(1, sq, skv, 8, 8, dim)
    nb = ih.ops.cross_attention_workspace(cd)
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device="cuda")
    captured("cross %d %d" % (sq, dim), lambda s: ih.ops.cross_attention(cd, q.data_ptr(), kv.data_ptr(), kv.data_ptr(), o.data_ptr(),
             d_workspace=ws.data_ptr(), workspace_bytes=nb, stream=s), o)
print("captures ok")
"""


def test_first_calls_may_be_captured():
    # A fresh process, whose first call of each kernel is under capture.
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(ih.__file__)))
    r = subprocess.run([sys.executable, "-W", "ignore", "-c", CHILD], env=env, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "captures ok" in r.stdout, r.stdout + r.stderr
