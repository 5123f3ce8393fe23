"""The operators of an fp8 half block, as a program calls them one by one: the norms before and after
a block with its gate and its residual's scale, the quantization of operands to e4m3 with a scale for
each block of 128 (behind a feed-forward's gated activation, or of a weight), and the linear layer on
such operands.

A case is a dict of plain values.  `listed` holds the fixed ones, `draw` one more of the same
ranges, `prepare` makes what a program has in hand before the call, `run` is one pass: the
operators in elementary torch operations, or with `own` the package's entry points.  `work` is the
bytes and operations a pass cannot do without, `exact` the same outputs in float64.

The widths are the package's configurations (1024 wide with 2816 hidden, 1280 with 3680); an utterance
has up to 750 latent frames (30 s), a text up to 256 tokens.  Codes are returned as e4m3 values beside
their scales.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1}
BLOCK = 128
MOST = 448.0  # the largest e4m3 value
LEAST = 2.0 ** -126  # of a scale
EPS = 1e-5


# ---- the cases ------------------------------------------------------------------------------
def _norm(rows, dim, dtype, stream=None, h=None, branch="none", norm="rms", has_branch=True, gate=False, mod=False, mod_rows=0,
          affine=True, stream_scale=1.0, branch_scale=1.0, **kw):
    """stream: the residual stream's type; h: the normed output's; branch, norm: the norm after the
    block and the one before the next; gate: by channel and group of mod_rows rows; mod: a scale and a
    shift likewise; affine: weights (and biases where a norm has a mean) by channel."""
    return dict(kw, kind="norm", rows=rows, dim=dim, dtype=dtype, stream=stream or dtype, h=h or dtype, branch=branch, norm=norm,
                has_branch=has_branch, gate=gate, mod=mod, mod_rows=mod_rows or rows, affine=affine, stream_scale=stream_scale,
                branch_scale=branch_scale)


def _quantize(rows, dim, dtype, gated=False, act="none", weight=False, **kw):
    """gated: act of the first half of each row times the second; weight: blocks of 128 x 128."""
    return dict(kw, kind="quantize", rows=rows, dim=dim, dtype=dtype, gated=gated, act=act, weight=weight)


def _linear(m, n, k, out, act="none", bias=True, gate_rows=0, residual=False, **kw):
    """gate_rows: rows that share a row of the gate (0: no gate)."""
    return dict(kw, kind="linear", m=m, n=n, k=k, out=out, act=act, bias=bias, gate_rows=gate_rows, residual=residual)


def listed():
    return [
        # One new token of four streams between two blocks: a latency.
        _norm(4, 1280, "bf16", branch="rms", branch_scale=0.5, name="norm_4_tokens"),
        # A text's states (an odd token count) before a block, in f32 with a mean.
        _norm(253, 1280, "f32", norm="layer", has_branch=False, name="norm_f32_text"),
        # Both guidance rows of a 30 s utterance: the block's output normed, gated and added to the f32 stream, the
        # next block's modulated input as fp8 operands.
        _norm(1500, 1024, "bf16", stream="f32", h="fp8", branch="rms", gate=True, mod=True, mod_rows=750, affine=True, name="norm_fp8_1500"),
        # 16 utterances with their guidance rows, 16-bit in and out around the f32 stream.
        _norm(24000, 1280, "bf16", stream="f32", norm="layer", gate=True, mod=True, mod_rows=750, affine=False, name="norm_batch"),
        # The gated activation of eight new tokens.
        _quantize(8, 2816, "bf16", gated=True, act="silu", name="quantize_8_tokens"),
        # A weight at load: W1 and W3 of a block.
        _quantize(5632, 1024, "f32", weight=True, name="quantize_weight"),
        # The gated activation of 16 utterances with their guidance rows.
        _quantize(24000, 2816, "bf16", gated=True, act="silu", name="quantize_batch"),
        # Four new tokens onto both halves of the widest hidden layer: the weights are all there is to read.
        _linear(4, 7360, 1280, "bf16", bias=False, name="linear_4_tokens"),
        # A text's states, the last block of K short.
        _linear(253, 1280, 1000, "f16", act="gelu", name="linear_text"),
        # The down projection of both guidance rows of a 30 s utterance: gated, onto the f32 stream.
        _linear(1500, 1024, 2816, "f32", gate_rows=750, residual=True, name="linear_gated_residual"),
        # The up projection of 16 utterances with their guidance rows.
        _linear(24000, 5632, 1024, "bf16", bias=False, name="linear_batch"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 250, 333, 512, 1000, 1024, 1280, 1536, 2816, 3680, 5632])
    if kind == "norm":
        gate = rng.random() < 0.5
        mod = rng.random() < 0.5
        mod_rows = rng.choice([1, 101, 750]) if gate or mod else 0
        # (The vectors of a modulation by row are read as the rows are.)
        rows = _log_int(rng, 1, 24000 * 1280 // max(dim, 1024) // ((2 if dtype == "f32" else 1) * (2 if mod_rows == 1 else 1)))
        return _norm(rows, dim, dtype, stream=rng.choice([dtype, "f32"]), h=rng.choice([dtype, "fp8"]),
                     branch=rng.choice(["none", "rms", "layer"]), norm=rng.choice(["rms", "layer"]), has_branch=rng.random() < 0.8,
                     gate=gate, mod=mod, mod_rows=mod_rows, affine=rng.random() < 0.6,
                     stream_scale=rng.choice([1.0, 1.0, 0.8]), branch_scale=rng.choice([1.0, 0.25]))
    if kind == "quantize":
        if rng.random() < 0.3:
            return _quantize(rng.choice([64, 333, 1024, 1280, 2816, 5632]), dim, dtype, weight=True)
        gated = rng.random() < 0.6
        rows = _log_int(rng, 1, 24000 * 2816 // max(dim, 1024) // (2 if dtype == "f32" else 1))
        return _quantize(rows, dim, dtype, gated=gated, act=rng.choice(["silu", "gelu", "gelu_tanh", "sigmoid"]) if gated else "none")
    n = rng.choice([64, 96, 333, 1000, 1024, 1280, 2816, 4096, 5632])
    k = rng.choice([64, 128, 250, 512, 1000, 1024, 1280, 2816, 3680])
    m = _log_int(rng, 1, 24000 * 5632 * 1024 // (max(n, 1024) * max(k, 1024)))
    residual = rng.random() < 0.4
    return _linear(m, n, k, rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.6, residual=residual,
                   act=rng.choice(["none", "none", "none", "relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"]),
                   gate_rows=rng.choice([1, 101, 750]) if residual and rng.random() < 0.5 else 0)


# ---- the inputs -----------------------------------------------------------------------------
def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _states(gen, rows, dim, dtype, std=1.0):
    """Activations: channels of different spread, a few of them far above the rest, and a mean."""
    spread = torch.exp(0.5 * torch.randn(dim, generator=gen, device=DEV))
    spread = torch.where(torch.rand(dim, generator=gen, device=DEV) < 0.01, spread * 16.0, spread)
    mean = 0.2 * torch.randn(dim, generator=gen, device=DEV)
    return ((torch.randn(rows, dim, generator=gen, device=DEV) * std + mean) * spread).to(dtype)


def _blocks(k):
    return -(-k // BLOCK)


def _block_max(v, rows):
    """The largest magnitude of each block of rows x 128: [ceil(r / rows), ceil(c / 128)]."""
    r, c = v.shape
    a = torch.nn.functional.pad(v.abs(), (0, _blocks(c) * BLOCK - c, 0, -r % rows))
    return a.reshape(-1, rows, _blocks(c), BLOCK).amax(dim=(1, 3))


def _spread(s, rows, r, c):
    """Each block's scale at the block's elements."""
    return s.repeat_interleave(rows, dim=0)[:r].repeat_interleave(BLOCK, dim=1)[:, :c]


def _plain_codes(v, rows):
    """e4m3 values and their scales of f32 values."""
    s = torch.clamp(_block_max(v, rows) / MOST, min=LEAST)
    return (v / _spread(s, rows, *v.shape)).to(torch.float8_e4m3fn), s


def _bytes(*shape):
    return torch.empty(*shape, dtype=torch.uint8, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = dict(case=case, plan=None)
    if case["kind"] == "norm":
        rows, dim = case["rows"], case["dim"]
        t, ts = TYPE[case["dtype"]], TYPE[case["stream"]]
        groups = -(-rows // case["mod_rows"])
        # The timestep's modulation holds every vector of a group side by side.
        mod = _randn(gen, groups, 3 * dim, std=0.3)
        bias = lambda kind: _randn(gen, dim, std=0.2) if case["affine"] and kind == "layer" else None  # noqa: E731
        weight = lambda on: 1.0 + _randn(gen, dim, std=0.2) if case["affine"] and on else None  # noqa: E731
        after = case["has_branch"] and case["branch"] != "none"
        st.update(x=_states(gen, rows, dim, ts), y=_states(gen, rows, dim, t, std=0.5) if case["has_branch"] else None,
                  gate=mod[:, :dim] if case["gate"] and case["has_branch"] else None,
                  scale=mod[:, dim:2 * dim] if case["mod"] else None, shift=mod[:, 2 * dim:] if case["mod"] else None,
                  wb=weight(after), bb=bias(case["branch"]) if after else None, w=weight(True), b=bias(case["norm"]),
                  x_out=torch.empty(rows, dim, dtype=ts, device=DEV) if case["has_branch"] else None)
        if case["h"] == "fp8":
            st.update(h=_bytes(rows, dim), hs=torch.empty(rows, _blocks(dim), device=DEV))
        else:
            st.update(h=torch.empty(rows, dim, dtype=t, device=DEV), hs=None)
        return st
    if case["kind"] == "quantize":
        rows, dim = case["rows"], case["dim"]
        t = TYPE[case["dtype"]]
        x = _randn(gen, rows, dim, dtype=t, std=dim ** -0.5) if case["weight"] else _states(gen, rows, dim * (2 if case["gated"] else 1), t)
        st.update(x=x, q=_bytes(rows, dim), s=torch.empty(-(-rows // (BLOCK if case["weight"] else 1)), _blocks(dim), device=DEV))
        return st
    m, n, k, to = case["m"], case["n"], case["k"], TYPE[case["out"]]
    x, xs = _plain_codes(_states(gen, m, k, torch.float32), 1)
    w, ws = _plain_codes(_randn(gen, n, k, std=k ** -0.5), BLOCK)
    st.update(x=x, xs=xs, w=w, ws=ws, bias=_randn(gen, n, std=0.5) if case["bias"] else None,
              gate=_randn(gen, -(-m // case["gate_rows"]), n, std=0.3) if case["gate_rows"] else None,
              residual=_randn(gen, m, n, dtype=to) if case["residual"] else None, y=torch.empty(m, n, dtype=to, device=DEV))
    return st


# ---- the operators in elementary operations ---------------------------------------------------
def _act(y, name):
    if name == "relu":
        return torch.clamp(y, min=0.0)
    if name == "silu":
        return y / (1.0 + torch.exp(-y))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-y))
    if name == "tanh":
        return torch.tanh(y)
    if name == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _normed(v, kind):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    return v if kind == "none" else v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS)


def _affine(v, w, b):
    v = v if w is None else v * w
    return v if b is None else v + b


def _plain_norm(st):
    case = st["case"]
    each = torch.arange(case["rows"], device=DEV) // case["mod_rows"]
    r = st["x"].float() * case["stream_scale"]
    out = {}
    if st["y"] is not None:
        y = _affine(_normed(st["y"].float(), case["branch"]), st["wb"], st["bb"]) * case["branch_scale"]
        r = r + (y if st["gate"] is None else y * st["gate"][each])
        out["x"] = r.to(TYPE[case["stream"]])
    h = _affine(_normed(r, case["norm"]), st["w"], st["b"])
    if st["scale"] is not None:
        h = h * (1.0 + st["scale"][each]) + st["shift"][each]
    if case["h"] == "fp8":
        out["h"], out["h_scale"] = _plain_codes(h, 1)
    else:
        out["h"] = h.to(TYPE[case["dtype"]])
    return out


def _plain_quantize(st):
    case = st["case"]
    v = st["x"].float()
    if case["gated"]:
        v = _act(v[:, :case["dim"]], case["act"]) * v[:, case["dim"]:]
    q, s = _plain_codes(v, BLOCK if case["weight"] else 1)
    return {"q": q, "s": s}


def _plain_linear(st):
    case = st["case"]
    m, n, k = case["m"], case["n"], case["k"]
    x = st["x"].float() * _spread(st["xs"], 1, m, k)
    w = st["w"].float() * _spread(st["ws"], BLOCK, n, k)
    y = torch.matmul(x, w.t())
    if st["bias"] is not None:
        y = y + st["bias"]
    y = _act(y, case["act"])
    if st["gate"] is not None:
        y = y * st["gate"].repeat_interleave(case["gate_rows"], dim=0)[:m]
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return {"y": y.to(TYPE[case["out"]])}


# ---- the package's entry points ---------------------------------------------------------------
def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "irodori-tts-burn_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import irodori_hip
    return irodori_hip


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _plan(st):
    """What a program makes once per shape: the call's description."""
    if st["plan"] is None:
        ih, case = _package(), st["case"]
        if case["kind"] == "norm":
            on = st["gate"] is not None or st["scale"] is not None
            desc = ih.BlockNormDesc(case["rows"], case["dim"], dtype=case["dtype"], stream_dtype=case["stream"], h_dtype=case["h"],
                                    branch_norm=case["branch"], norm=case["norm"], branch_eps=EPS, eps=EPS,
                                    stream_scale=case["stream_scale"], branch_scale=case["branch_scale"],
                                    mod_rows=case["mod_rows"] if on else 0, ldm=3 * case["dim"])
        elif case["kind"] == "quantize":
            desc = ih.BlockQuantizeDesc(case["rows"], case["dim"], dtype=case["dtype"], gated=case["gated"], activation=case["act"],
                                        block_rows=BLOCK if case["weight"] else 1)
        else:
            desc = ih.LinearFp8Desc(case["m"], case["n"], case["k"], out_dtype=case["out"], activation=case["act"],
                                    gate_rows=case["gate_rows"])
        st["plan"] = (ih.ops, desc)
    return st["plan"]


def _own(st):
    ops, desc = _plan(st)
    kind, stream = st["case"]["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "norm":
        ops.block_norm(desc, _ptr(st["x"]), d_branch=_ptr(st["y"]), d_branch_weight=_ptr(st["wb"]), d_branch_bias=_ptr(st["bb"]),
                       d_gate=_ptr(st["gate"]), d_x_out=_ptr(st["x_out"]), d_weight=_ptr(st["w"]), d_bias=_ptr(st["b"]),
                       d_scale=_ptr(st["scale"]), d_shift=_ptr(st["shift"]), d_h=_ptr(st["h"]), d_h_scales=_ptr(st["hs"]), stream=stream)
        out = {} if st["y"] is None else {"x": st["x_out"]}
        if st["hs"] is None:
            out["h"] = st["h"]
        else:
            out["h"], out["h_scale"] = st["h"].view(torch.float8_e4m3fn), st["hs"]
        return out
    if kind == "quantize":
        ops.block_quantize(desc, _ptr(st["x"]), _ptr(st["q"]), _ptr(st["s"]), stream=stream)
        return {"q": st["q"].view(torch.float8_e4m3fn), "s": st["s"]}
    ops.linear_fp8(desc, _ptr(st["x"]), _ptr(st["xs"]), _ptr(st["w"]), _ptr(st["ws"]), _ptr(st["y"]), d_bias=_ptr(st["bias"]),
                   d_gate=_ptr(st["gate"]), d_residual=_ptr(st["residual"]), stream=stream)
    return {"y": st["y"]}


def run(st):
    if own:
        return _own(st)
    return {"norm": _plain_norm, "quantize": _plain_quantize, "linear": _plain_linear}[st["case"]["kind"]](st)


# ---- the work, and the outputs in float64 -------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        n = case["rows"] * case["dim"]
        groups, after = -(-case["rows"] // case["mod_rows"]), case["has_branch"] and case["branch"] != "none"
        vectors = groups * ((1 if case["gate"] and case["has_branch"] else 0) + (2 if case["mod"] else 0))
        if case["affine"]:
            vectors += 1 + (case["norm"] == "layer") + (after + (after and case["branch"] == "layer"))
        nbytes = n * (SIZE[case["stream"]] + SIZE[case["h"]]) + 4 * vectors * case["dim"]
        if case["has_branch"]:
            nbytes += n * (SIZE[case["dtype"]] + SIZE[case["stream"]])
        if case["h"] == "fp8":
            nbytes += 4 * case["rows"] * _blocks(case["dim"])
        return {"bytes": nbytes, "flops": n * (16 if case["has_branch"] else 8)}
    if case["kind"] == "quantize":
        n = case["rows"] * case["dim"]
        scales = -(-case["rows"] // BLOCK) if case["weight"] else case["rows"]
        return {"bytes": n * (SIZE[case["dtype"]] * (2 if case["gated"] else 1) + 1) + 4 * scales * _blocks(case["dim"]),
                "flops": n * (8 if case["gated"] else 3)}
    m, n, k, eo = case["m"], case["n"], case["k"], SIZE[case["out"]]
    nbytes = (m + n) * k + 4 * _blocks(k) * (m + -(-n // BLOCK)) + m * n * eo * (2 if case["residual"] else 1)
    if case["bias"]:
        nbytes += 4 * n
    if case["gate_rows"]:
        nbytes += 4 * n * -(-m // case["gate_rows"])
    return {"bytes": nbytes, "flops": 2 * m * n * k}


def _exact_codes(v, tall):
    """The unrounded quotients and the scales of blocks of 128 columns, a row or 128 rows tall."""
    r, c = v.shape
    scales = torch.zeros(-(-r // tall), -(-c // BLOCK), dtype=torch.float64, device=DEV)
    q = torch.empty_like(v)
    for j in range(scales.shape[1]):
        cols = slice(j * BLOCK, min(c, (j + 1) * BLOCK))
        top = v[:, cols].abs().max(dim=1).values
        if tall > 1:
            top = torch.stack([part.max() for part in top.split(tall)])
        scales[:, j] = torch.maximum(top / MOST, torch.full_like(top, LEAST))
        q[:, cols] = v[:, cols] / scales[torch.arange(r, device=DEV) // tall, j][:, None]
    return q, scales


_EXACT_ACT = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
              "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        group = torch.div(torch.arange(case["rows"], device=DEV), case["mod_rows"], rounding_mode="floor")

        def norm(v, kind, w, b):
            if kind == "rms":
                v = v / (v.pow(2).sum(1, keepdim=True) / case["dim"] + EPS).sqrt()
            elif kind == "layer":
                v = (v - v.sum(1, keepdim=True) / case["dim"]) / (v.var(1, correction=0, keepdim=True) + EPS).sqrt()
            if w is not None:
                v = v * w.double()
            return v if b is None else v + b.double()

        r, res = case["stream_scale"] * st["x"].double(), {}
        if st["y"] is not None:
            g = 1.0 if st["gate"] is None else st["gate"].double()[group]
            r = r + case["branch_scale"] * g * norm(st["y"].double(), case["branch"], st["wb"], st["bb"])
            res["x"] = r
        h = norm(r, case["norm"], st["w"], st["b"])
        if st["scale"] is not None:
            h = h + h * st["scale"].double()[group] + st["shift"].double()[group]
        if case["h"] == "fp8":
            res["h"], res["h_scale"] = _exact_codes(h, 1)
        else:
            res["h"] = h
        return res
    if case["kind"] == "quantize":
        v = st["x"].double()
        if case["gated"]:
            a, b = v.chunk(2, dim=1)
            v = _EXACT_ACT[case["act"]](a) * b
        q, s = _exact_codes(v, BLOCK if case["weight"] else 1)
        return {"q": q, "s": s}
    m, n, k = case["m"], case["n"], case["k"]
    y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
    for j in range(_blocks(k)):  # block by block of the reduction
        cols = slice(j * BLOCK, min(k, (j + 1) * BLOCK))
        by_row = st["ws"][:, j].double()[torch.arange(n, device=DEV) // BLOCK]
        y += (st["x"][:, cols].double() @ st["w"][:, cols].double().T) * st["xs"][:, j, None].double() * by_row[None]
    if st["bias"] is not None:
        y += st["bias"].double()
    y = _EXACT_ACT[case["act"]](y)
    if st["gate"] is not None:
        y *= st["gate"].double()[torch.arange(m, device=DEV) // case["gate_rows"]]
    if st["residual"] is not None:
        y += st["residual"].double()
    return {"y": y}
