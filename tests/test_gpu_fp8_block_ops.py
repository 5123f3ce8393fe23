"""The operators of an fp8 half block (norms around a block, quantization to e4m3 blocks of 128, linear layer on
them) on the GPU against float64 formulas of the same rounded inputs, one by one and as the feed-forward half
block they make up.

Tolerances are bounds of each element's error, from the arithmetic: u = eps / 2 of the output's type for its
rounding, F = 2^-24 for each f32 step; an e4m3 code is off by at most 2^-4 of its value, or 2^-10 below 2^-6.
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
LEAST = 2.0 ** -126


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


def blocks(n):
    return -(-n // 128)


def close(got, ref, tol, what=""):
    got = got.double()
    err = (got - ref).abs()
    bad = ~(err <= tol)  # a NaN is bad
    if bad.any():
        i = int((err / tol).nan_to_num(nan=math.inf).flatten().argmax())
        raise AssertionError("%s: %d of %d off, worst at %d: got %r want %r tol %r" % (
            what, int(bad.sum()), bad.numel(), i, got.flatten()[i].item(), ref.flatten()[i].item(), tol.flatten()[i].item()))


def padded(r, c, pad, dtype, offset=0, fill=math.nan):
    """A [r, c] view with pad elements between its rows, and the flat tensor it lies in."""
    t = TYPE.get(dtype, torch.uint8)
    flat = torch.full((r * (c + pad) + offset + 64,), fill if t != torch.uint8 else 0x7f, dtype=t, device="cuda")
    return flat, flat[offset:offset + r * (c + pad)].view(r, c + pad)[:, :c]


def outside(flat, r, c, pad, offset=0):
    """What lies around such a view."""
    kept = torch.ones_like(flat, dtype=torch.bool)
    kept[offset:offset + r * (c + pad)].view(r, c + pad)[:, :c] = False
    return flat[kept]


def block_max(v, tall=1):
    r, c = v.shape
    p = torch.nn.functional.pad(v, (0, blocks(c) * 128 - c, 0, -r % tall))
    return p.reshape(-1, tall, blocks(c), 128).amax(dim=(1, 3))


def spread(s, shape, tall=1):
    return s.repeat_interleave(tall, 0)[:shape[0]].repeat_interleave(128, 1)[:, :shape[1]]


def values(q):
    return q.view(torch.float8_e4m3fn).double()


def close_codes(q, s, ref, tol, what="", tall=1):
    """Codes and scales against float64 values known to tol."""
    top, slack = block_max(ref.abs(), tall) / 448, block_max(tol, tall) / 448
    top = top.clamp(min=LEAST)
    close(s, top, slack + F * (top + slack), what + " scales")
    full = spread(s.double(), ref.shape, tall)
    close(values(q) * full, ref, torch.maximum((ref.abs() + tol) * 2.0 ** -4, full * 2.0 ** -10) + 1.01 * tol + 2 * F * ref.abs(), what)


# ---- norms around a block ---------------------------------------------------------------------
def norm_ref(v, kind, eps, err):
    """The float64 norm of rows known to err, and its bound: sums of at most 32 in order, then 16 more, in f32."""
    n = v.shape[1]
    if kind == "none":
        return v, err
    d = v - v.mean(1, keepdim=True) if kind == "layer" else v
    r = 1 / (d.square().mean(1, keepdim=True) + eps).sqrt()
    y = d * r
    # f32: the differences and the mean that they miss, the squares' sum (half of its relative error), root and quotient.
    tol = F * (40 * y.abs() + (64 if kind == "layer" else 0))
    return y, tol + r * (err + err.mean(1, keepdim=True)) + y.abs() * r * (y.abs() * err).mean(1, keepdim=True)


class Norms:
    def __init__(self, rows, dim, dtype, stream_dtype=None, h=None, branch="none", norm="rms", has_branch=True, gate=False, mod=False,
                 mod_rows=0, affine=True, a=1.0, c=1.0, eps=1e-5, beps=1e-5, pad=0, offset=0, seed=1, x_out=True, std=1.0):
        st, h = stream_dtype or dtype, h or dtype
        self.kw = dict(branch=branch, norm=norm, a=a, c=c, eps=eps, beps=beps, mod_rows=mod_rows or rows)
        self.types = dtype, st, h
        self.geometry = rows, dim, pad, offset
        self.xflat, self.x = padded(rows, dim, pad, st, offset)
        self.x.copy_(randn(seed, rows, dim, dtype=st, std=std))
        self.y = None
        if has_branch:
            _, self.y = padded(rows, dim, pad, dtype, offset)
            self.y.copy_(randn(seed + 1, rows, dim, dtype=dtype) * 3 + 1)
        groups = -(-rows // (mod_rows or rows))
        m = randn(seed + 2, groups, 3 * dim + 5, std=0.5)
        self.gate = m[:, :dim] if gate else None
        self.scale, self.shift = (m[:, dim:2 * dim], m[:, 2 * dim:3 * dim]) if mod else (None, None)
        w = randn(seed + 3, 4, dim)
        self.wb, self.bb = (w[0], w[1]) if affine and has_branch else (None, None)
        self.w, self.b = (w[2], w[3]) if affine else (None, None)
        self.xoflat, self.x_out = padded(rows, dim, pad, st, offset, CANARY) if x_out else (None, None)
        self.hflat, self.h = padded(rows, dim, pad, h, offset, CANARY)
        self.sflat, self.hs = padded(rows, blocks(dim), pad, "f32", offset, CANARY) if h == "fp8" else (None, None)
        any_mod = gate or mod
        self.desc = ih.BlockNormDesc(rows, dim, dtype=dtype, stream_dtype=st, h_dtype=h, branch_norm=branch, norm=norm, branch_eps=beps,
                                     eps=eps, stream_scale=a, branch_scale=c, mod_rows=self.kw["mod_rows"] if any_mod else 0, ldx=dim + pad,
                                     ldb=dim + pad, ldxo=dim + pad, ldh=dim + pad, ldhs=blocks(dim) + pad, ldm=m.stride(0))

    def __call__(self):
        ih.ops.block_norm(self.desc, ptr(self.x), ptr(self.y), ptr(self.wb), ptr(self.bb), ptr(self.gate), ptr(self.x_out), ptr(self.w),
                          ptr(self.b), ptr(self.scale), ptr(self.shift), ptr(self.h), ptr(self.hs), stream=stream())

    def reference(self):
        k = self.kw
        each = torch.arange(self.x.shape[0], device="cuda") // k["mod_rows"]
        one = torch.ones((), dtype=torch.float64, device="cuda")
        x = self.x.double()
        r, err = k["a"] * x, F * (k["a"] * x).abs()
        if self.y is not None:
            y, e = norm_ref(self.y.double(), k["branch"], k["beps"], torch.zeros_like(x))
            wb, bb = (one if self.wb is None else self.wb.double()), (one * 0 if self.bb is None else self.bb.double())
            g = k["c"] * (one if self.gate is None else self.gate.double()[each])
            t = y * wb + bb
            e = (e * wb.abs() + 4 * F * ((y * wb).abs() + bb.abs())) * g.abs()
            r = r + g * t
            err = err + e + 2 * F * (g * t).abs() + F * r.abs()
        h, e = norm_ref(r, k["norm"], k["eps"], err)
        w, b = (one if self.w is None else self.w.double()), (one * 0 if self.b is None else self.b.double())
        s, d = (one * 0, one * 0) if self.scale is None else (self.scale.double()[each], self.shift.double()[each])
        out = (h * w + b) * (1 + s) + d
        mag = ((h * w).abs() + b.abs()) * (1 + s.abs()) + d.abs()
        return r, err, out, e * (w * (1 + s)).abs() + 8 * F * mag

    def check(self, what=""):
        dtype, st, h = self.types
        r, err, out, e = self.reference()
        if self.x_out is not None:
            close(self.x_out, r, err + u(st) * (r.abs() + err) + tiny(st), what + " x_out")
        if h == "fp8":
            close_codes(self.h, self.hs, out, e, what + " h")
        else:
            close(self.h, out, e + u(h) * (out.abs() + e) + tiny(h), what + " h")
        rows, dim, pad, off = self.geometry
        assert (outside(self.hflat, rows, dim, pad, off) == (0x7f if h == "fp8" else CANARY)).all()
        if self.x_out is not None:
            assert (outside(self.xoflat, rows, dim, pad, off) == CANARY).all()
        if h == "fp8":
            assert (outside(self.sflat, rows, blocks(dim), pad, off) == CANARY).all()


DIMS = [1, 7, 64, 127, 130, 250, 333, 512, 520, 1001, 1024, 1280, 1536, 1601, 2048, 2056, 2816, 4096, 4099, 5632, 6144, 8200, 16384]


@pytest.mark.parametrize("dtype,st", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("h", ["same", "fp8"])
@pytest.mark.parametrize("dim", DIMS)
def test_block_norm(dtype, st, h, dim):
    n = Norms(5, dim, dtype, st, dtype if h == "same" else h, branch="rms", norm="layer", gate=True, mod=True, mod_rows=2, a=0.75, c=0.5)
    n()
    n.check()


@pytest.mark.parametrize("branch", ["none", "rms", "layer"])
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("h", ["bf16", "fp8"])
@pytest.mark.parametrize("affine,gate,mod", [(False, False, False), (True, False, False), (False, True, False), (False, False, True), (True, True, True)])
def test_block_norm_parts(branch, norm, h, affine, gate, mod):
    for dim in (200, 2500):
        n = Norms(3, dim, "bf16", "f32", h, branch=branch, norm=norm, affine=affine, gate=gate, mod=mod, mod_rows=1)
        n()
        n.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", ["same", "fp8"])
@pytest.mark.parametrize("rows", [1, 2, 4, 67, 1501])
def test_block_norm_without_a_branch(dtype, h, rows):
    n = Norms(rows, 330, dtype, "f32", dtype if h == "same" else h, has_branch=False, norm="rms", x_out=rows == 4, mod=True, mod_rows=50)
    n()
    n.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", ["same", "fp8"])
@pytest.mark.parametrize("dim,pad,offset", [(40, 3, 1), (333, 1, 3), (1280, 8, 0), (2049, 3, 1)])
def test_block_norm_strides_and_alignment(dtype, h, dim, pad, offset):
    """Rows apart and off every wide boundary; what lies between them is neither read (NaN there) nor written."""
    n = Norms(6, dim, dtype, dtype, dtype if h == "same" else h, branch="layer", norm="rms", gate=True, mod_rows=3, pad=pad, offset=offset)
    n()
    n.check()


@pytest.mark.parametrize("dim", [96, 2300])
def test_block_norm_onto_its_stream(dim):
    n = Norms(9, dim, "bf16", "f32", "fp8", branch="rms", norm="rms")
    ref = n.reference()
    n.x_out, n.xoflat = n.x, n.xflat
    n()
    close(n.x, ref[0], ref[1] + F * ref[0].abs() + tiny("f32"))
    close_codes(n.h, n.hs, ref[2], ref[3])


def test_block_norm_one_output_alone():
    n = Norms(4, 300, "bf16", "f32", branch="rms", norm="layer", affine=False)
    n.h.fill_(CANARY)
    h, n.h = n.h, None
    n()
    r, err, _, _ = n.reference()
    close(n.x_out, r, err + F * r.abs() + tiny("f32"))
    assert (h == CANARY).all()
    m = Norms(4, 300, "bf16", "f32", branch="rms", norm="layer", affine=False, x_out=False)
    m()
    m.check()


def test_block_norm_broadcast_stream():
    # A stride of 0 repeats one row of the stream, of the branch and of the modulation.
    n = Norms(1, 384, "bf16", branch="rms", gate=True, mod=True, seed=9)
    rows = 5
    d = ih.BlockNormDesc(rows, 384, dtype="bf16", branch_norm="rms", mod_rows=1, ldx=0, ldb=0, ldm=0)
    xo, h = (torch.empty(rows, 384, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ih.ops.block_norm(d, ptr(n.x), ptr(n.y), ptr(n.wb), ptr(n.bb), ptr(n.gate), ptr(xo), ptr(n.w), ptr(n.b), ptr(n.scale), ptr(n.shift), ptr(h),
                      stream=stream())
    n()
    n.check()
    assert (xo == n.x_out).all() and (h == n.h).all()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dim", [130, 3000])
@pytest.mark.parametrize("mean,std", [(0.0, 1e25), (0.0, 1e-12), (3e4, 1.0), (0.0, 1e18), (1e30, 1e26), (-2e38, 3e37)])
def test_block_norm_of_extreme_rows(kind, dim, mean, std):
    """Squares past f32's range, means far above the spread, rows far below eps."""
    x = randn(3, 4, dim) * std + mean
    n = Norms(4, dim, "f32", norm=kind, has_branch=False, affine=False, x_out=False)
    n.x.copy_(x)
    n()
    n.check("%s %g %g" % (kind, mean, std))


def test_block_norm_constant_rows():
    # No spread: (v - mean) is 0, and eps alone is under the root.
    for v in (0.0, 1.0, -3.3e4, 2.0 ** 100):
        n = Norms(2, 777, "f32", norm="layer", has_branch=False, affine=False, x_out=False)
        n.x.fill_(v)
        n()
        assert (n.h == 0).all(), v


@pytest.mark.parametrize("dim", [2, 1024, 4096])
def test_block_norm_constant_rows_whose_sum_passes_the_range(dim):
    # (Sums of a power of two of powers of two are exact, so the differences are 0.)
    for v in (2.0 ** 126, -(2.0 ** 127), 2.0 ** 127):
        n = Norms(2, dim, "f32", norm="layer", has_branch=False, x_out=False)
        n.x.fill_(v)
        n()
        assert (n.h == n.b).all(), v


@pytest.mark.parametrize("eps", [1e-5, 1e-30])
@pytest.mark.parametrize("dim", [3, 250, 777, 1000, 2048, 2816, 5632, 16384])
def test_block_norm_constant_rows_far_from_zero(dim, eps):
    """Constants of any mantissa, a row each: their sums round, and yet the differences from the mean are all 0."""
    g = torch.Generator().manual_seed(dim)
    v = torch.exp(torch.empty(400).uniform_(math.log(1e-3), math.log(3e38), generator=g)) * (1 - 2 * torch.randint(0, 2, (400,), generator=g))
    v[:6] = torch.tensor([9.90373153e14, 7.56785854e14, 8e11, 1e18, -3.3e9, 1.7e10])
    for dtype in ("f32", "bf16"):
        n = Norms(400, dim, dtype, norm="layer", has_branch=False, affine=False, x_out=False, eps=eps)
        n.x.copy_(v[:, None].to(TYPE[dtype]).expand(-1, dim))
        n()
        assert (n.h == 0).all(), n.x[(n.h != 0).any(1), 0].tolist()[:8]
    m = Norms(400, dim, "bf16", "f32", branch="layer", norm="none", affine=False, x_out=False, beps=eps)  # the branch's norm: r = x
    m.x.zero_()
    m.y.copy_(v[:, None].to(torch.bfloat16).expand(-1, dim))
    m()
    assert (m.h == 0).all()


@pytest.mark.parametrize("dim", [3, 250, 1000, 2816, 16384])
@pytest.mark.parametrize("few", [0.001, 0.2, 0.5])
def test_block_norm_rows_within_a_few_steps_of_a_constant(dim, few):
    """Rows of a constant and its f32 neighbours: all of the spread is in the last bits.

    The differences from the rounded mean are whole numbers of half steps d, those of the mean at most half a step, so
    that mean(d)^2 <= var: E d^2 <= 2 var and E |d| <= 1.5 s.  A sum has at most 48 roundings in a row, so mean(d) is off by 48 F 1.5 s = 72 F s;
    the variance by 50 F E d^2 + 2 mean(d) 72 F s + 2 F var <= 246 F var, its root by half of that, and 3 F of quotient and product."""
    g = torch.Generator().manual_seed(dim)
    v = torch.exp(torch.empty(300, 1).uniform_(math.log(1e3), math.log(1e36), generator=g)) * (1 - 2 * torch.randint(0, 2, (300, 1), generator=g))
    steps = torch.where(torch.rand(300, dim, generator=g) < few, torch.randint(-2, 3, (300, dim), generator=g), torch.zeros((), dtype=torch.long))
    x = (v.view(torch.int32) + steps.int()).view(torch.float32).cuda()
    n = Norms(300, dim, "f32", norm="layer", has_branch=False, affine=False, x_out=False, eps=1e-20)
    n.x.copy_(x)
    n()
    away = x.double() - x.double()[:, :1]  # exact
    y, _ = norm_ref(away, "layer", 1e-20, torch.zeros_like(away))
    close(n.h, y, F * (126 * y.abs() + 72) + u("f32") * y.abs(), "steps")


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dim", [1000, 5632, 16384])
def test_block_norm_keeps_a_large_eps_where_squares_pass_the_range(kind, dim):
    # The least rows whose squares' sum is infinite in f32: there an eps of 1e30 is 5e-5 of the mean square at 16384 columns.
    sign = 1 - 2 * (torch.arange(dim, device="cuda") % 2)
    for factor in (1.01, 1.5, 30.0):
        n = Norms(3, dim, "f32", norm=kind, has_branch=False, affine=False, x_out=False, eps=1e30)
        n.x.copy_((sign * factor * math.sqrt(2.0 ** 128 / dim)).float().expand(3, -1))
        n()
        n.check("%s %g" % (kind, factor))


@pytest.mark.parametrize("dim", [256, 2304])
def test_block_norm_specials_stay_in_their_row(dim):
    n = Norms(5, dim, "bf16", "f32", "fp8", branch="rms", norm="rms", affine=False)
    clean = Norms(5, dim, "bf16", "f32", "fp8", branch="rms", norm="rms", affine=False)
    clean()
    n.x[1, 5] = math.inf
    n.y[3, 7] = math.nan
    n()
    for row in (0, 2, 4):
        assert torch.equal(n.h[row], clean.h[row]) and torch.equal(n.hs[row], clean.hs[row]) and torch.equal(n.x_out[row], clean.x_out[row])
    # v / sqrt(inf): the infinity itself is NaN, the rest 0.
    h = values(n.h)
    assert h[1, 5].isnan() and (h[1, :5] == 0).all() and (h[1, 6:] == 0).all() and h[3].isnan().all()
    assert n.x_out[1, 5] == math.inf and torch.isfinite(n.x_out[1, 6:]).all()


# ---- quantization -----------------------------------------------------------------------------
def run_quantize(x, dim, dtype, q, s, **kw):
    d = ih.BlockQuantizeDesc(x.shape[0], dim, dtype=dtype, ldx=x.stride(0), ldq=q.stride(0), lds=s.stride(0), **kw)
    ih.ops.block_quantize(d, ptr(x), ptr(q), ptr(s), stream=stream())


def codes_ref(x, tall=1):
    """The definition in f32 on the CPU, whose quotients are correctly rounded."""
    v = x.float().cpu()
    a = torch.where(v.abs() < math.inf, v.abs(), torch.zeros(()))
    s = (block_max(a, tall) / 448).clamp(min=LEAST)
    q = v / spread(s, v.shape, tall)
    q = torch.where(v.abs() < math.inf, q, torch.full((), math.nan))
    return q.to(torch.float8_e4m3fn).view(torch.uint8), s


def same_codes(q, ref):
    q, ref = q.cpu(), ref
    both = ((q & 0x7f) == 0x7f) & ((ref & 0x7f) == 0x7f)  # NaN of either sign
    assert ((q == ref) | both).all(), int(((q != ref) & ~both).sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tall", [1, 128])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 250), (130, 333), (257, 1000), (300, 2816), (1, 16000), (1000, 64), (2049, 40)])
def test_block_quantize_is_exact(dtype, tall, rows, dim):
    x = randn(1, rows, dim, dtype=dtype)
    x *= torch.exp(2 * randn(2, rows, 1)).to(x.dtype)
    q, s = torch.full((rows, dim), 0x7f, dtype=torch.uint8, device="cuda"), torch.empty(-(-rows // tall), blocks(dim), device="cuda")
    run_quantize(x, dim, dtype, q, s, block_rows=tall)
    rq, rs = codes_ref(x, tall)
    assert torch.equal(s.cpu(), rs)
    same_codes(q, rq)


def test_block_quantize_ties_and_limits():
    """Every e4m3 value and every midpoint, scaled so that the quotients are those numbers exactly, and scales whose
    reciprocal is rounded either way."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mids = (codes[:-1] + codes[1:]) / 2
    for k, factor in enumerate([1.0, 0.75, 1.5, 1.0 / 3, 7.0, 2.0 ** -100, 1.2345e-5, 3.7e30, 2.0 ** -126, 2.0 ** -117]):
        f = torch.tensor(factor)
        rows = []
        for part in (codes, mids, -mids):
            row = torch.zeros(128)
            row[:part.numel()] = part * f
            row[127] = 448 * f
            rows.append(row)
        x = torch.stack(rows).cuda()
        q, s = torch.zeros(3, 128, dtype=torch.uint8, device="cuda"), torch.empty(3, 1, device="cuda")
        run_quantize(x, 128, "f32", q, s)
        rq, rs = codes_ref(x)
        assert torch.equal(s.cpu(), rs), factor
        same_codes(q, rq)


@pytest.mark.parametrize("factor", [1.2345 * 2.0 ** -126, 1.9 * 2.0 ** -126, 1.1 * 2.0 ** -125, 1.7 * 2.0 ** -122, 1.3 * 2.0 ** -112, 1.9 * 2.0 ** -104,
                                    1.6 * 2.0 ** -95, 1.45 * 2.0 ** -93, 1.3 * 2.0 ** -65, 1.3 * 2.0 ** -64, 1.7 * 2.0 ** -63, 1.2 * 2.0 ** -20, 1.55, 1.3 * 2.0 ** 118])
def test_block_quantize_next_to_midpoints(factor):
    """Values at and a step beside the midpoints of two codes, under scales of any mantissa down to the least: rows quantized one by
    one, tile by tile, and behind a norm that passes its rows on."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mids = ((codes[:-1] + codes[1:]) / 2).double()
    g = torch.Generator().manual_seed(3)
    rows = []
    for i in range(300):
        top = torch.tensor(448 * factor * (1 + 0.001 * i if factor < 2.0 ** 118 else 1), dtype=torch.float32)
        s = (top / 448).double()
        row = (mids * s).float()[torch.randperm(126, generator=g)]
        step = torch.randint(-1, 2, (126,), generator=g, dtype=torch.int32)
        row = (row.view(torch.int32) + step).view(torch.float32) * (1 - 2 * torch.randint(0, 2, (126,), generator=g))
        rows.append(torch.cat([row, torch.zeros(1), top[None]]))
    x = torch.stack(rows).cuda()
    q, s = torch.zeros(300, 128, dtype=torch.uint8, device="cuda"), torch.empty(300, 1, device="cuda")
    rq, rs = codes_ref(x)
    run_quantize(x, 128, "f32", q, s)
    assert torch.equal(s.cpu(), rs)
    same_codes(q, rq)
    q.zero_()
    d = ih.BlockNormDesc(300, 128, dtype="f32", h_dtype="fp8", norm="none")
    ih.ops.block_norm(d, ptr(x), d_h=ptr(q), d_h_scales=ptr(s), stream=stream())
    assert torch.equal(s.cpu(), rs)
    same_codes(q, rq)
    for i in (0, 7, 299):  # (a tile has one scale)
        t = x[i:i + 1].contiguous()
        run_quantize(t, 128, "f32", q[i:i + 1], s[i:i + 1], block_rows=128)
        assert torch.equal(s[i].cpu(), rs[i])
        same_codes(q[i], rq[i])


def test_block_quantize_largest_of_many_blocks():
    # The largest magnitude's quotient may round to above 448: its code is 448 all the same.
    x = randn(7, 4096, 128) * torch.exp(8 * randn(8, 4096, 1))
    q, s = torch.zeros(4096, 128, dtype=torch.uint8, device="cuda"), torch.empty(4096, 1, device="cuda")
    run_quantize(x, 128, "f32", q, s)
    v = values(q)
    assert torch.isfinite(v).all() and (v.abs().amax(1) == 448).all()


@pytest.mark.parametrize("tall", [1, 128])
def test_block_quantize_specials(tall):
    x = randn(3, 130, 300)
    x[0, :128] = 0.0
    x[1, 5], x[2, 130], x[2, 131], x[3, 299] = math.inf, -math.inf, math.nan, math.nan
    x[4, :128] = 1e-40  # below the least scale's codes
    x[5, 128:256] = math.nan
    x[6, 128:256] = -math.inf
    q, s = torch.zeros(130, 300, dtype=torch.uint8, device="cuda"), torch.empty(-(-130 // tall), 3, device="cuda")
    run_quantize(x, 300, "f32", q, s, block_rows=tall)
    rq, rs = codes_ref(torch.where(x.isnan(), torch.full((), math.inf, device="cuda"), x), tall)  # (a NaN counts for no maximum)
    assert torch.equal(s.cpu(), rs) and torch.isfinite(s).all()
    same_codes(q, rq)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [True, False])
def test_block_quantize_activations(dtype, act, gated):
    acts = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
            "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}
    rows, dim = 37, 200
    x = randn(1, rows, dim * (2 if gated else 1), dtype=dtype, std=2.0)
    q, s = torch.zeros(rows, dim, dtype=torch.uint8, device="cuda"), torch.empty(rows, 2, device="cuda")
    run_quantize(x, dim, dtype, q, s, gated=gated, activation=act)
    a = x[:, :dim].double()
    ref = acts[act](a)
    # The activations' own error is a few F of the argument and of 1; the product one more.
    tol = 16 * F * (a.abs() + 1) if act != "none" else torch.zeros_like(a)
    if gated:
        g = x[:, dim:].double()
        ref, tol = ref * g, tol * g.abs() + F * (ref * g).abs()
    close_codes(q, s, ref, tol, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tall,gated", [(1, False), (1, True), (128, False)])
@pytest.mark.parametrize("rows,dim,pad,offset", [(3, 40, 3, 1), (140, 333, 1, 3), (5, 1280, 8, 0)])
def test_block_quantize_strides_and_alignment(dtype, tall, gated, rows, dim, pad, offset):
    wide = dim * (2 if gated else 1)
    _, x = padded(rows, wide, pad, dtype, offset)
    x.copy_(randn(1, rows, wide, dtype=dtype))
    qf, q = padded(rows, dim, pad, "u8", offset)
    sr = -(-rows // tall)
    sf, s = padded(sr, blocks(dim), pad, "f32", offset, CANARY)
    run_quantize(x, dim, dtype, q, s, block_rows=tall, gated=gated)
    v = x.float()
    rq, rs = codes_ref(v[:, :dim] * v[:, dim:] if gated else v, tall)
    assert torch.equal(s.cpu(), rs)
    same_codes(q, rq)
    assert (outside(qf, rows, dim, pad, offset) == 0x7f).all() and (outside(sf, sr, blocks(dim), pad, offset) == CANARY).all()


def test_block_quantize_repeats_itself():
    # Blocks of what the codes stand for: the same codes and scales.
    x = randn(1, 64, 512)
    q, s = torch.zeros(64, 512, dtype=torch.uint8, device="cuda"), torch.empty(64, 4, device="cuda")
    run_quantize(x, 512, "f32", q, s)
    y = (values(q) * spread(s.double(), (64, 512))).float()
    q2, s2 = torch.zeros_like(q), torch.empty_like(s)
    run_quantize(y, 512, "f32", q2, s2)
    # 448 s rounded to f32, over 448: s to two roundings; a code is at most 2^-4 from a midpoint.
    assert torch.equal(q, q2) and ((s - s2).abs() <= 2 * F * s).all()


# ---- linear layer -----------------------------------------------------------------------------
ACTS = {
    "none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
    "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
}


def operands(m, n, k, seed=1, pad=0, offset=0):
    """Any finite codes, and scales of any sign and size around 2^-6."""
    g = torch.Generator().manual_seed(seed)
    def codes(r):
        c = torch.randint(0, 254, (r, k), generator=g)
        _, v = padded(r, k, pad, "u8", offset)
        v.copy_((c + (c >= 127)).to(torch.uint8).cuda())  # neither NaN
        return v
    def scales(r):
        _, v = padded(r, blocks(k), pad, "f32", offset if pad else 0)
        v.copy_((torch.randn(r, blocks(k), generator=g) * 2.0 ** -6).cuda())
        return v
    return codes(m), scales(m), codes(n), scales(blocks(n))


def run_linear(x, xs, w, ws, y, out, act="none", bias=None, gate=None, gate_rows=0, residual=None, m=None):
    d = ih.LinearFp8Desc(m or x.shape[0], w.shape[0], x.shape[1], out_dtype=out, activation=act, gate_rows=gate_rows, ldx=x.stride(0),
                         ldw=w.stride(0), ldy=y.stride(0), ldr=residual.stride(0) if residual is not None else None, ldxs=xs.stride(0),
                         ldws=ws.stride(0))
    ih.ops.linear_fp8(d, ptr(x), ptr(xs), ptr(w), ptr(ws), ptr(y), d_bias=ptr(bias), d_gate=ptr(gate), d_residual=ptr(residual), stream=stream())


def linear_ref(x, xs, w, ws, out, act="none", bias=None, gate=None, gate_rows=0, residual=None):
    """Float64 result and its tolerance: products of two codes have 8 bits; a sum of k of them loses at most 2 F each of their
    magnitudes, truncated; a block's scale and its addition 3 F; the rest as in the linear operator of wider types.  For 16-bit
    outputs of more than 16 rows the matrix cores align 8 products to the largest of them, p, and drop what lies below 2^-13 p of the 7
    others: less than 7 / 8 2^-10 p, at most that of the 8 magnitudes' sum."""
    m, k = x.shape
    xv = values(x) * spread(xs.double(), x.shape)
    wv = values(w) * spread(ws.double(), w.shape, 128)
    z, mag = xv @ wv.T, xv.abs() @ wv.abs().T
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    y = ACTS[act](z)
    aligned = 2.0 ** -10 if out != "f32" and m > 16 else 0.0
    tol = 1.13 * (aligned + (2 * min(k, 128) + 3 * blocks(k) + 8) * F) * mag + (16 * F * (z.abs() + 1) if act != "none" else 0)
    if gate is not None:
        g = gate.double()[torch.arange(m, device="cuda") // gate_rows]
        y, tol = y * g, (tol + F * y.abs()) * g.abs()
    if residual is not None:
        y = y + residual.double()
        tol = tol + F * y.abs()
    return y, tol + u(out) * (y.abs() + tol) + tiny(out)


SHAPES = [(1, 1, 1), (1, 1024, 512), (2, 96, 2816), (3, 5, 7), (4, 3680, 1280), (15, 64, 250), (16, 300, 64), (16, 100, 5000), (17, 33, 65),
          (32, 64, 64), (64, 128, 1000), (65, 1280, 192), (101, 333, 1001), (253, 1280, 1280), (300, 520, 96), (1500, 1024, 128),
          (1100, 2050, 72), (40, 70, 130), (700, 1500, 252), (2100, 4000, 68), (5000, 5632, 64), (6100, 5632, 1024), (1900, 1300, 135),
          (130, 260, 384), (200, 140, 640), (90, 90, 900), (1500, 1024, 2816), (260, 2500, 3680)]


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_fp8(out, m, n, k):
    ops = operands(m, n, k)
    bias, res = randn(3, n), randn(4, m, n, dtype=out)
    gate = randn(5, -(-m // 7), n)
    y = torch.full((m, n), CANARY, dtype=TYPE[out], device="cuda")
    run_linear(*ops, y, out)
    close(y, *linear_ref(*ops, out), "plain")
    run_linear(*ops, y, out, "silu", bias=bias, gate=gate, gate_rows=7, residual=res)
    close(y, *linear_ref(*ops, out, "silu", bias, gate, 7, res), "all")
    # onto the residual
    ref = linear_ref(*ops, out, "none", bias, None, 0, res)
    run_linear(*ops, res, out, bias=bias, residual=res)
    close(res, *ref, "in place")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m", [2, 70])
def test_linear_fp8_activations(act, m):
    x, xs, w, ws = operands(m, 40, 64)
    xs *= 2.0 ** -3
    y = torch.empty(m, 40, device="cuda")
    run_linear(x, xs, w, ws, y, "f32", act)
    close(y, *linear_ref(x, xs, w, ws, "f32", act), act)


@pytest.mark.parametrize("m,n,k", [(1, 65, 40), (5, 24, 333), (40, 70, 129), (130, 260, 128), (70, 300, 1300)])
@pytest.mark.parametrize("pad,offset", [(16, 0), (4, 4), (3, 0), (3, 1), (2, 2), (1, 3)])
def test_linear_fp8_strides_and_alignment(m, n, k, pad, offset):
    """Rows apart and off every wide boundary; what lies between and around them is neither read into
    the result (NaN there) nor written."""
    ops = operands(m, n, k, pad=pad, offset=offset)
    flat, y = padded(m, n, pad, "bf16", offset, CANARY)
    run_linear(*ops, y, "bf16")
    close(y, *linear_ref(*ops, "bf16"), "strided")
    assert (outside(flat, m, n, pad, offset) == CANARY).all()


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k,pad", [(1003, 1283, 1288, 8), (403, 2819, 2824, 8), (1501, 1291, 128, 8), (2101, 2051, 72, 8),
                                       (1501, 5635, 3688, 8), (1902, 1801, 136, 3), (6203, 5635, 260, 4)])
def test_linear_fp8_edges_of_large_tiles(out, m, n, k, pad):
    """Tiles that end past the last row and inside a lane's columns, everything after the product with them, onto the
    residual; the columns between rows keep what they hold."""
    ops = operands(m, n, k, pad=pad)
    bias, gate = randn(3, n), randn(5, -(-m // 7), n)
    flat, y = padded(m, n, pad, out, 0, CANARY)
    y.copy_(randn(4, m, n, dtype=out))
    ref = linear_ref(*ops, out, "silu", bias, gate, 7, y.clone())
    run_linear(*ops, y, out, "silu", bias=bias, gate=gate, gate_rows=7, residual=y)
    close(y, *ref, "edges")
    assert (outside(flat, m, n, pad) == CANARY).all()


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", [(4090, 4090, 900), (9000, 2900, 388), (650, 2816, 520), (8191, 4092, 1100), (5100, 5632, 128), (6100, 5632, 132)])
def test_linear_fp8_tiles_one_after_another(out, m, n, k):
    """Workgroups that take several tiles, one load ahead of the products across them, with one block of K or an odd or even
    number, whole and cut; inner tiles and edges; each part of the epilogue."""
    ops = operands(m, n, k)
    bias, gate, res = randn(3, n), randn(5, -(-m // 7), n), randn(4, m, n, dtype=out)
    y = torch.full((m, n), CANARY, dtype=TYPE[out], device="cuda")
    run_linear(*ops, y, out)
    close(y, *linear_ref(*ops, out), "plain")
    run_linear(*ops, y, out, "tanh", bias=bias)
    close(y, *linear_ref(*ops, out, "tanh", bias), "bias")
    ref = linear_ref(*ops, out, "none", None, gate, 7, res)
    run_linear(*ops, res, out, gate=gate, gate_rows=7, residual=res)
    close(res, *ref, "gated residual")


@pytest.mark.parametrize("m", [5, 40, 300])
def test_linear_fp8_broadcast_rows(m):
    # A stride of 0 repeats one row of x, of its scales and of the residual; shorter strides than k overlap.
    x, xs, w, ws = operands(1, 200, 384)
    res = randn(3, 1, 200, dtype="bf16")
    y = torch.empty(m, 200, dtype=torch.bfloat16, device="cuda")
    d = ih.LinearFp8Desc(m, 200, 384, ldx=0, ldxs=0, ldr=0)
    ih.ops.linear_fp8(d, ptr(x), ptr(xs), ptr(w), ptr(ws), ptr(y), d_residual=ptr(res), stream=stream())
    close(y, *linear_ref(x.expand(m, -1).contiguous(), xs.expand(m, -1), w, ws, "bf16", residual=res.expand(m, -1)))
    long = operands(1, 1, 384 + 128 * m)[0][0]
    xs = operands(m, 1, 384)[1]
    d = ih.LinearFp8Desc(m, 200, 384, ldx=128)
    ih.ops.linear_fp8(d, ptr(long), ptr(xs), ptr(w), ptr(ws), ptr(y), stream=stream())
    close(y, *linear_ref(torch.stack([long[128 * i:128 * i + 384] for i in range(m)]), xs, w, ws, "bf16"))


@pytest.mark.parametrize("m,n", [(9, 300), (70, 300), (600, 2600)])
def test_linear_fp8_specials_stay_in_their_rows(m, n):
    k = 400
    ops = operands(m, n, k)
    x, xs, w, ws = ops
    clean = torch.empty(m, n, device="cuda")
    run_linear(*ops, clean, "f32")
    x[2, 399], xs[4, 1], w[n - 1, 3] = 0x7f, math.inf, 0xff
    xs[6, 0] = 0.0
    y = torch.empty(m, n, device="cuda")
    run_linear(*ops, y, "f32")
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[2], bad[4], bad[:, n - 1] = True, True, True
    assert not torch.isfinite(y[bad]).any()
    bad[6] = True
    assert torch.equal(y[~bad], clean[~bad])
    ref, tol = linear_ref(x, xs, w, ws, "f32")
    close(y[6, :n - 1], ref[6, :n - 1], tol[6, :n - 1])


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("m,n", [(9, 300), (70, 300), (600, 1000), (1500, 1024), (6100, 2816), (24000, 1024)])
def test_linear_fp8_specials_stay_in_their_rows_of_16_bits(out, m, n):
    # (Of the last two a workgroup takes several tiles: none keeps anything of the one before it.)
    k = 400
    x, xs, w, ws = operands(m, n, k)
    clean, y = (torch.empty(m, n, dtype=TYPE[out], device="cuda") for _ in range(2))
    run_linear(x, xs, w, ws, clean, out)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    x[m - 2, 399], xs[4, 1], w[n - 1, 3] = 0x7f, math.inf, 0xff
    bad[m - 2], bad[4], bad[:, n - 1] = True, True, True
    for i in range(130, m - 2, 260):
        x[i, i % k] = 0x7f
        bad[i] = True
    run_linear(x, xs, w, ws, y, out)
    assert not torch.isfinite(y[bad]).any()
    assert torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (9, 300, 700), (16, 130, 5000), (40, 70, 130), (70, 300, 1300), (130, 260, 384), (600, 1000, 400), (1500, 1024, 520),
                                   (101, 333, 1001), (1100, 2050, 71), (6100, 2816, 260), (12000, 1280, 264), (9000, 2900, 388), (8191, 4092, 600)])
def test_linear_fp8_scales_whose_product_leaves_the_range(out, m, n, k):
    """Scales whose product is no normal f32 number though the term is one, in every third row between ordinary rows and rows of
    zero scales, behind a gate and onto a residual as well.  A subnormal product is off by 2^-150, times a block's sum of at most 128 448^2 <
    2^25; sums that are subnormal round to 2^-150, one a block."""
    x, xs, w, ws = operands(m, n, k)
    mant = lambda s: torch.where(s < 0, -1.0, 1.0) * (1 + (s.abs() * 4096) % 1)  # noqa: E731
    power = lambda e: torch.tensor(2.0, dtype=torch.float64, device="cuda") ** e  # noqa: E731
    gate, res = 1 + randn(5, -(-m // 7), n, std=0.1), randn(4, m, n, dtype=out)
    for e_x, e_w in ((-70, -70), (-76, -76), (-100, -40), (-126, -15), (-149, 10), (64, 64), (66, 66), (126, 3), (20, 110)):
        a, b, s = x, w, mant(xs)
        s[0::3] = (s[0::3] * power(e_x)).float()
        s[1::3] = (s[1::3] * power(-6)).float()
        s[2::3] = 0.0
        t = (mant(ws) * power(e_w)).float()
        if e_x > 0:  # no more than 4 of the least products a block, and rows and columns of zeros of either sign
            a = torch.where(torch.arange(k, device="cuda") % 37 == 3, x & 0x81, x & 0x80)
            a[6::12] &= 0x80
            b = w & 0x81
            b[5::9] &= 0x80
            b[n // 2:n // 2 + 128] &= 0x80
        what = "2^%d 2^%d" % (e_x, e_w)
        lost = blocks(k) * (2.0 ** -150 + (2.0 ** -125 if e_x < 0 else 0))
        y = torch.full((m, n), CANARY, dtype=TYPE[out], device="cuda")
        run_linear(a, s, b, t, y, out)
        ref, tol = linear_ref(a, s, b, t, out)
        close(y, ref, tol + lost, what)
        y = res.clone()
        ref, tol = linear_ref(a, s, b, t, out, "none", None, gate, 7, res)
        run_linear(a, s, b, t, y, out, gate=gate, gate_rows=7, residual=y)
        close(y, ref, tol + 2 * lost, what + " onto the residual")


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", [(9, 300, 700), (40, 70, 130), (70, 300, 1300), (600, 1000, 400), (1500, 1024, 520), (101, 333, 1001), (6100, 2816, 260),
                                   (12000, 1280, 264), (9000, 2900, 388)])
def test_linear_fp8_rows_beside_scales_out_of_range(out, m, n, k):
    """Rows whose own scales are ordinary hold the same bits whatever their neighbours' are, everything after the product with them."""
    x, xs, w, ws = operands(m, n, k)
    xs, ws = xs * 2.0 ** -60, ws * 2.0 ** 60
    bias, gate, res = randn(3, n), randn(5, -(-m // 7), n), randn(4, m, n, dtype=out)
    clean, y = (torch.empty(m, n, dtype=TYPE[out], device="cuda") for _ in range(2))
    for act in ("none", "silu"):
        for kw in (dict(), dict(bias=bias, gate=gate, gate_rows=7, residual=res)):
            run_linear(x, xs, w, ws, clean, out, act, **kw)
            far = xs.clone()
            far[1::3, 0] = 2.0 ** 110
            run_linear(x, far, w, ws, y, out, act, **kw)
            for i in (0, 2):
                assert torch.equal(y[i::3], clean[i::3]), (act, len(kw), i)


@pytest.mark.parametrize("channels", [1.0, 16.0])
@pytest.mark.parametrize("m,n,k", [(16, 300, 1000), (64, 64, 1000), (300, 520, 900), (253, 1280, 250), (113, 333, 1001), (1500, 1024, 1024), (6100, 2816, 400),
                                   (24000, 1024, 250), (12000, 1280, 900)])
def test_linear_fp8_bits_of_16_bit_outputs(m, n, k, channels):
    """The products' own error, apart from the output's rounding: the residual takes the rounded result away, and what is left is rounded to
    2^-11 of at most 2^-11 of it.  Of each 8 neighbouring products a part below 2^-13 of the largest one's power of two is lost, of a sign of its own;
    where no bit lies there, nothing is; up to 16 rows nothing at all.  `channels`: every 16th column of x as many times the rest."""
    wide = torch.where(torch.arange(k, device="cuda") % 16 == 5, channels, 1.0)
    x, w = randn(1, m, k) * wide, randn(2, n, k, std=k ** -0.5)
    xq, xs = torch.empty(m, k, dtype=torch.uint8, device="cuda"), torch.empty(m, blocks(k), device="cuda")
    wq, ws = torch.empty(n, k, dtype=torch.uint8, device="cuda"), torch.empty(blocks(n), blocks(k), device="cuda")
    run_quantize(x, k, "f32", xq, xs)
    run_quantize(w, k, "f32", wq, ws, block_rows=128)
    ref, _ = linear_ref(xq, xs, wq, ws, "f32")
    y = -ref.to(torch.float16)
    want = ref + y.double()
    run_linear(xq, xs, wq, ws, y, "f16", residual=y)
    rows, cols = torch.arange(0, m, -(-m // 64), device="cuda"), torch.arange(0, n, -(-n // 64), device="cuda")
    err = (y.double() - want)[rows][:, cols]
    lost = torch.zeros((), dtype=torch.float64, device="cuda")
    for b in range(blocks(k) if m > 16 else 0):
        part = lambda q: torch.nn.functional.pad(values(q[:, 128 * b:128 * b + 128]), (0, -(k - 128 * b) % 8 if b == blocks(k) - 1 else 0))  # noqa: E731
        p = (part(xq[rows])[:, None] * part(wq[cols])[None]).unflatten(2, (-1, 8))
        step = torch.exp2(torch.floor(torch.log2(p.abs().amax(3, keepdim=True).clamp(min=2.0 ** -20))) - 13)
        f = xs[rows, b].double()[:, None] * ws[cols // 128, b].double()[None]
        lost += ((torch.remainder(p.abs(), step) != 0) * step.square()).sum(dim=(2, 3)).mul(f.square()).sum()
    # f32: as in linear_ref, most of it 2 F of the magnitudes in a row, roundings of independent signs.
    size = ref[rows][:, cols].norm()
    got = float(err.norm() / size)
    assert got <= float(lost.sqrt() / size) + 2.0 ** -22 + 4 * F * math.sqrt(k / 8)


@pytest.mark.parametrize("m", [4, 40, 300])
def test_linear_fp8_rows_far_apart(m):
    # Rows of x, w, y and the scales some 2^27 bytes apart or more: offsets past 32 bits.
    k, n, step = 130, 130, (1 << 32) // m + 64
    buf = torch.empty(m * step + k, dtype=torch.uint8, device="cuda")
    xc, xsc, w, ws = operands(m, n, k)
    x = torch.as_strided(buf, (m, k), (step, 1))
    x.copy_(xc)
    y = torch.empty(m, n, device="cuda")
    run_linear(x, xsc, w, ws, y, "f32")
    close(y, *linear_ref(xc, xsc, w, ws, "f32"), "x")
    del x
    f = buf.view(torch.uint8)[:(buf.numel() // 4) * 4].view(torch.float32)
    xs = torch.as_strided(f, (m, 2), (step // 4, 1))
    xs.copy_(xsc)
    run_linear(xc, xs, w, ws, y, "f32")
    close(y, *linear_ref(xc, xsc, w, ws, "f32"), "x scales")
    yf = torch.as_strided(f, (m, n), (step // 4, 1))
    run_linear(xc, xsc, w, ws, yf, "f32")
    close(yf, *linear_ref(xc, xsc, w, ws, "f32"), "y")


@pytest.mark.parametrize("m", [3, 50, 200])
def test_linear_fp8_long_reduction(m):
    k = (1 << 22) + 132 if m == 50 else 100004
    ops = operands(m, 40, k)
    y = torch.empty(m, 40, device="cuda")
    run_linear(*ops, y, "f32")
    close(y, *linear_ref(*ops, "f32"))


# ---- together ---------------------------------------------------------------------------------
class FeedForward:
    """x + gate * rms(W2 (silu(W1 h) * W3 h)), h = rms(x) modulated: an fp8 half block and the next one's operands."""

    def __init__(self, rows, dim, hidden, dtype, mod_rows):
        self.shape = rows, dim, hidden, dtype, mod_rows
        cast = lambda w: self.quantize(w)  # noqa: E731
        self.w13, self.w13s = cast(randn(11, 2 * hidden, dim, std=dim ** -0.5))
        self.w2, self.w2s = cast(randn(12, dim, hidden, std=hidden ** -0.5))
        self.norms = 1 + 0.1 * randn(13, 3, dim)
        self.mod = randn(14, -(-rows // mod_rows), 3 * dim, std=0.3)
        b = lambda r, c: torch.empty(r, c, dtype=torch.uint8, device="cuda")  # noqa: E731
        s = lambda r, c: torch.empty(r, blocks(c), device="cuda")  # noqa: E731
        self.h, self.hs, self.u, self.us, self.next, self.nexts = b(rows, dim), s(rows, dim), b(rows, hidden), s(rows, hidden), b(rows, dim), s(rows, dim)
        self.a = torch.empty(rows, 2 * hidden, dtype=TYPE[dtype], device="cuda")
        self.y = torch.empty(rows, dim, dtype=TYPE[dtype], device="cuda")
        common = dict(dtype=dtype, stream_dtype="f32", h_dtype="fp8", mod_rows=mod_rows, ldm=3 * dim)
        self.before = ih.BlockNormDesc(rows, dim, **common)
        self.after = ih.BlockNormDesc(rows, dim, branch_norm="rms", **common)
        self.up = ih.LinearFp8Desc(rows, 2 * hidden, dim, out_dtype=dtype)
        self.act = ih.BlockQuantizeDesc(rows, hidden, dtype=dtype, gated=True, activation="silu")
        self.down = ih.LinearFp8Desc(rows, dim, hidden, out_dtype=dtype)

    @staticmethod
    def quantize(w):
        q, s = torch.empty(w.shape, dtype=torch.uint8, device="cuda"), torch.empty(blocks(w.shape[0]), blocks(w.shape[1]), device="cuda")
        run_quantize(w, w.shape[1], "f32", q, s, block_rows=128)
        return q, s

    def __call__(self, x):
        st, dim = stream(), self.shape[1]
        gate, scale, shift = (ptr(self.mod) + 4 * dim * i for i in range(3))
        ih.ops.block_norm(self.before, ptr(x), d_weight=ptr(self.norms[0]), d_scale=scale, d_shift=shift, d_h=ptr(self.h), d_h_scales=ptr(self.hs), stream=st)
        ih.ops.linear_fp8(self.up, ptr(self.h), ptr(self.hs), ptr(self.w13), ptr(self.w13s), ptr(self.a), stream=st)
        ih.ops.block_quantize(self.act, ptr(self.a), ptr(self.u), ptr(self.us), stream=st)
        ih.ops.linear_fp8(self.down, ptr(self.u), ptr(self.us), ptr(self.w2), ptr(self.w2s), ptr(self.y), stream=st)
        ih.ops.block_norm(self.after, ptr(x), ptr(self.y), d_branch_weight=ptr(self.norms[1]), d_gate=gate, d_x_out=ptr(x), d_weight=ptr(self.norms[2]),
                          d_scale=scale, d_shift=shift, d_h=ptr(self.next), d_h_scales=ptr(self.nexts), stream=st)

    def reference(self, x):
        rows, dim, hidden, _, mod_rows = self.shape
        each = torch.arange(rows, device="cuda") // mod_rows
        gate, scale, shift = self.mod.double()[each].split(dim, 1)
        rms = lambda v: v / (v.square().mean(1, keepdim=True) + 1e-5).sqrt()  # noqa: E731
        n = self.norms.double()
        h = rms(x.double()) * n[0] * (1 + scale) + shift
        a = h @ (values(self.w13) * spread(self.w13s.double(), self.w13.shape, 128)).T
        v = torch.nn.functional.silu(a[:, :hidden]) * a[:, hidden:]
        y = v @ (values(self.w2) * spread(self.w2s.double(), self.w2.shape, 128)).T
        inc = gate * rms(y) * n[1]
        return inc, rms(x.double() + inc) * n[2] * (1 + scale) + shift


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,hidden,mod_rows", [(1, 256, 640, 1), (75, 256, 704, 25), (300, 1024, 2816, 150)])
def test_feed_forward_half_block(dtype, rows, dim, hidden, mod_rows):
    blk = FeedForward(rows, dim, hidden, dtype, mod_rows)
    x = randn(20, rows, dim)
    inc, nxt = blk.reference(x)
    y = x.clone()
    blk(y)
    # e4m3 roundings of h and of the gated product, each at most 2^-4 of an element (2^-10 of a scale, below); a relative error
    # d of h gives the two factors of the gated product at most (1.1 + 1) d of their own norm together on independent elements, silu's
    # slope being at most 1.1; roundings to the 16-bit type are far below.  The norm after it passes the relative error on.
    d = 2.0 ** -4
    assert (y.double() - x.double() - inc).norm() <= (2.1 * d + d + 8 * u(dtype)) * inc.norm()
    got = values(blk.next) * spread(blk.nexts.double(), nxt.shape)
    assert (got - nxt).norm() <= (d + (3.1 * d + 8 * u(dtype)) * float(inc.norm() / (x.double() + inc).norm()) * 2) * nxt.norm()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_feed_forward_captured_and_on_another_stream(dtype):
    """Captured from the first call on a stream of its own, replayed between eager work, against eager calls bit for bit; two
    blocks on two streams at once."""
    shape = (150, 256, 704, dtype, 75)
    blk, other = FeedForward(*shape), FeedForward(*shape)
    x0 = randn(20, 150, 256)
    x = x0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        blk(x)
    want = x0.clone()
    other(want)
    for i in range(4):
        x.copy_(x0)
        graph.replay()
        y = x0.clone()
        other(y)
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, want)
        assert torch.equal(blk.next, other.next) and torch.equal(blk.nexts, other.nexts)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    a, c = x0.clone(), x0.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        blk(a)
    with torch.cuda.stream(s2):
        other(c)
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

p = lambda t: t.data_ptr()
u8 = lambda *s: torch.randint(0, 126, s, device="cuda", dtype=torch.uint8)
for m, n, k in ((3, 64, 64), (40, 64, 64), (600, 512, 128), (1500, 1024, 2816), (12000, 5632, 1024), (40, 64, 33), (900, 2000, 130)):
    x, w, y = u8(m, k), u8(n, k), torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    xs, ws = torch.rand(m, -(-k // 128), device="cuda"), torch.rand(-(-n // 128), -(-k // 128), device="cuda")
    d = ih.LinearFp8Desc(m, n, k)
    captured("linear %d" % m, lambda s: ih.ops.linear_fp8(d, p(x), p(xs), p(w), p(ws), p(y), stream=s), y)
for dim, h in ((300, "bf16"), (3000, "fp8"), (1280, "fp8")):
    x = torch.randn(9, dim, device="cuda")
    b = torch.randn(9, dim, device="cuda").to(torch.bfloat16)
    xo, ho = torch.empty_like(x), torch.empty(9, dim, device="cuda", dtype=torch.bfloat16 if h == "bf16" else torch.uint8)
    hs = torch.empty(9, -(-dim // 128), device="cuda")
    d = ih.BlockNormDesc(9, dim, stream_dtype="f32", h_dtype=h, branch_norm="rms")
    captured("norm %d" % dim, lambda s: ih.ops.block_norm(d, p(x), p(b), d_x_out=p(xo), d_h=p(ho), d_h_scales=p(hs) if h == "fp8" else 0, stream=s), xo, ho)
for kw in (dict(), dict(gated=True, activation="silu"), dict(block_rows=128)):
    x = torch.randn(200, 600, device="cuda")
    q, s_ = torch.empty(200, 300, dtype=torch.uint8, device="cuda"), torch.empty(200, 3, device="cuda")
    d = ih.BlockQuantizeDesc(200, 300, dtype="f32", ldx=600, **kw)
    captured("quantize", lambda s: ih.ops.block_quantize(d, p(x), p(q), p(s_), stream=s), q, s_)
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
