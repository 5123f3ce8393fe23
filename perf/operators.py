"""The operators of a cross-attention half block, as a program calls them one by one: a linear
layer with its bias, activation, gate and residual in the product's epilogue, the rotary
positions of queries and keys, and attention from one sequence to an encoder's states of another
length.

A case is a dict of plain values.  `listed` holds the fixed ones, `draw` one more of the same
ranges, `prepare` makes what a program has in hand before the call, `run` is one pass: the
operators in elementary torch operations, or with `own` the package's entry points.  `work` is the
bytes and operations a pass cannot do without, `exact` the same outputs in float64.

The widths are the package's configurations (1024 / 16 heads / 2816, 1280 / 20 heads / 3680, the
1280-wide text encoder with 10 heads of 128); an utterance has up to 750 latent frames (30 s), a
text up to 256 tokens, a reference up to 375 frames.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases ------------------------------------------------------------------------------
def _linear(m, n, k, dtype, out=None, act="none", bias=True, gate_rows=0, residual=False, **kw):
    """gate_rows: rows that share a row of the gate (0: no gate); out: the output's type."""
    return dict(kw, kind="linear", m=m, n=n, k=k, dtype=dtype, out=out or dtype, act=act, bias=bias,
                gate_rows=gate_rows, residual=residual)


def _rope(batch, seq, heads, kv_heads, dim, dtype, layout="interleaved", rot_dim=None, rot_heads=None, scaling="none",
          factor=1.0, theta=10000.0, far=0, ragged=False, inverse=False, **kw):
    """rot_heads: heads that rotate, the others pass through (None: all); far: positions lie in
    [0, far) (0: 0 .. seq - 1); ragged: rows of several lengths."""
    return dict(kw, kind="rope", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, layout=layout,
                rot_dim=rot_dim or dim, rot_heads=heads if rot_heads is None else rot_heads, scaling=scaling,
                factor=factor, theta=theta, far=far, ragged=ragged, inverse=inverse)


def _cross(batch, sq, skv, heads, kv_heads, dim, dtype, ragged=False, masked=False, fused=False, **kw):
    """ragged: encoder states of several lengths; masked: keys dropped inside them, and the last
    row's condition dropped as a whole; fused: keys and values are halves of one projection."""
    return dict(kw, kind="cross", batch=batch, sq=sq, skv=skv, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                ragged=ragged, masked=masked, fused=fused)


def listed():
    return [
        # The conditioning layer on one timestep vector: a latency.
        _linear(1, 1024, 512, "bf16", act="silu", name="linear_vector"),
        # Four vectors onto the widest hidden layer: the weights are all there is to read.
        _linear(4, 3680, 1280, "f16", act="gelu_tanh", name="linear_4_rows"),
        # A text's states, as an f32 program projects them (an odd token count).
        _linear(253, 1280, 1280, "f32", act="gelu", name="linear_f32_text"),
        # The attention's output projection of both guidance rows of a 30 s utterance: gated, onto the f32 residual stream.
        _linear(1500, 1024, 1024, "bf16", out="f32", gate_rows=750, residual=True, name="linear_gated_residual"),
        # The up projection of 16 utterances with their guidance rows.
        _linear(24000, 5632, 1024, "bf16", act="silu", bias=False, name="linear_batch"),
        # One new token of eight streams, each at a position of its own in a long context.
        _rope(8, 1, 16, 4, 128, "bf16", layout="halves", rot_dim=64, scaling="by_parts", factor=8.0, far=262144, name="rope_token"),
        # Queries and keys of both guidance rows, half of the heads rotating, as the f32 model has them.
        _rope(2, 750, 16, 16, 64, "f32", rot_heads=8, name="rope_f32_750"),
        # Long packed texts of several lengths.
        _rope(8, 4001, 20, 20, 64, "bf16", layout="halves", scaling="ntk", factor=4.0, ragged=True, name="rope_long"),
        # One new token of eight streams against long references, heads shared four to one.
        _cross(8, 1, 8200, 16, 4, 128, "bf16", ragged=True, fused=True, name="cross_token"),
        # A short f32 request: 101 latent frames to 37 tokens of text.
        _cross(2, 101, 37, 16, 16, 64, "f32", masked=True, name="cross_f32_101x37"),
        # Both guidance rows of a 30 s utterance to the text and reference states.
        _cross(2, 750, 631, 16, 16, 64, "bf16", ragged=True, masked=True, fused=True, name="cross_750x631"),
        # 16 utterances with their guidance rows to long references.
        _cross(32, 750, 4100, 20, 20, 64, "f16", ragged=True, name="cross_batch"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "rope", "cross"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "linear":
        n = rng.choice([64, 96, 333, 1000, 1024, 1280, 2816, 3680, 4096, 5632])
        k = rng.choice([32, 250, 512, 1001, 1024, 1280, 2816, 3680])
        m = _log_int(rng, 1, 24000 * 5632 * 1024 // (max(n, 1024) * max(k, 1024)) // (8 if dtype == "f32" else 1))
        residual = rng.random() < 0.4
        return _linear(m, n, k, dtype, out=rng.choice([dtype, "f32"]), bias=rng.random() < 0.7, residual=residual,
                       act=rng.choice(["none", "none", "relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"]),
                       gate_rows=rng.choice([1, 101, 750]) if residual and rng.random() < 0.5 else 0)
    if kind == "rope":
        dim = rng.choice([64, 64, 128, 80, 256])
        heads = rng.choice([1, 10, 16, 20])
        batch = rng.randint(1, 8)
        return _rope(batch, _log_int(rng, 1, 8 * 4001 // (batch * (dim // 64))), heads, rng.choice([1, heads]), dim, dtype,
                     layout=rng.choice(["interleaved", "halves"]), rot_dim=rng.choice([dim, dim, dim // 2]),
                     rot_heads=rng.choice([heads, heads, (heads + 1) // 2]), scaling=rng.choice(["none", "linear", "ntk", "by_parts"]),
                     factor=rng.choice([2.0, 4.0, 8.0]), theta=rng.choice([10000.0, 500000.0]), far=rng.choice([0, 0, 65536, 1048576]),
                     ragged=rng.random() < 0.4, inverse=rng.random() < 0.3)
    dim = rng.choice([64, 64, 128])
    heads, kv_heads = rng.choice([(16, 16), (20, 20), (10, 10), (16, 4), (20, 5), (8, 1)])
    skv = _log_int(rng, 1, 16400)
    batch = rng.choice([1, 2, 3, 8, 32])
    most = 32 * 750 * 4100 * 20 * 64 // (skv * batch * heads * dim) // (8 if dtype == "f32" else 1)
    sq = rng.choice([1, 1, _log_int(rng, 1, 4000), _log_int(rng, 1, 4000)])
    return _cross(batch, max(1, min(sq, most)), skv, heads, kv_heads, dim, dtype, ragged=rng.random() < 0.5,
                  masked=rng.random() < 0.5, fused=rng.random() < 0.5)


def _lengths(batch, most):
    """The lengths of a ragged batch: the first row's is the longest, the others' spread over 0.3 to 1 of it."""
    return [max(1, int(most * (1.0 - 0.7 * ((0.618034 * b) % 1.0)))) for b in range(batch)]


# ---- the inputs -----------------------------------------------------------------------------
def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    t = TYPE[case["dtype"]]
    st = dict(case=case, plan=None)
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st.update(x=_randn(gen, m, k, dtype=t), w=_randn(gen, n, k, dtype=t, std=k ** -0.5),
                  bias=_randn(gen, n, std=0.5) if case["bias"] else None,
                  gate=_randn(gen, -(-m // case["gate_rows"]), n, std=0.3) if case["gate_rows"] else None,
                  residual=_randn(gen, m, n, dtype=TYPE[case["out"]]) if case["residual"] else None,
                  y=torch.empty(m, n, dtype=TYPE[case["out"]], device=DEV))
        return st
    if case["kind"] == "rope":
        b, s, h, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
        # Queries and keys are parts of one projection [b, s, heads + 2 kv_heads, dim].
        qkv = _randn(gen, b, s, h + 2 * hk, d, dtype=t)
        st.update(q=qkv[:, :, :h], k=qkv[:, :, h:h + hk], positions=None, lengths=None,
                  # Rows past a length stay as they were.
                  q_out=torch.zeros(b, s, h, d, dtype=t, device=DEV), k_out=torch.zeros(b, s, hk, d, dtype=t, device=DEV))
        if case["far"]:
            first = torch.randint(0, max(1, case["far"] - s), (b, 1), generator=gen, device=DEV)
            st["positions"] = (first + torch.arange(s, device=DEV)).to(torch.int32)
        if case["ragged"]:
            st["lengths"] = torch.tensor(_lengths(b, s), dtype=torch.int32, device=DEV)
        return st
    b, sq, skv, h, hk, d = (case[x] for x in ("batch", "sq", "skv", "heads", "kv_heads", "dim"))
    q = _randn(gen, b, sq, h, d, dtype=t)
    if case["fused"]:
        kv = _randn(gen, b, skv, 2, hk, d, dtype=t)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:
        k, v = _randn(gen, b, skv, hk, d, dtype=t), _randn(gen, b, skv, hk, d, dtype=t)
    st.update(q=q, k=k, v=v, lengths=None, mask=None, out=torch.empty(b, sq, h, d, dtype=t, device=DEV))
    if case["ragged"]:
        st["lengths"] = torch.tensor(_lengths(b, skv), dtype=torch.int32, device=DEV)
    if case["masked"]:
        mask = (torch.rand(b, skv, generator=gen, device=DEV) < 0.9).to(torch.uint8)
        mask[:, 0] = 1
        if b > 1:
            mask[-1] = 0
        st["mask"] = mask
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


def _plain_linear(st):
    case = st["case"]
    y = torch.matmul(st["x"].float(), st["w"].float().t())
    if st["bias"] is not None:
        y = y + st["bias"]
    y = _act(y, case["act"])
    if st["gate"] is not None:
        y = y * st["gate"].repeat_interleave(case["gate_rows"], dim=0)[:case["m"]]
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return {"y": y.to(TYPE[case["out"]])}


# A pair turns this many times over the trained length: above the first it keeps its frequency,
# below the second its positions are divided by the factor, between them it moves from one to the other.
BETA_FAST, BETA_SLOW, TRAINED = 32.0, 1.0, 4096.0


def _frequencies(case):
    """Radians per position of each pair, float64."""
    rot = case["rot_dim"]
    theta = case["theta"]
    if case["scaling"] == "ntk":
        theta = theta * case["factor"] ** (rot / (rot - 2.0))
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    f = torch.exp(i * (-2.0 / rot * math.log(theta)))
    if case["scaling"] == "linear":
        f = f / case["factor"]
    elif case["scaling"] == "by_parts":
        turns = TRAINED * f / (2.0 * math.pi)
        keep = torch.clamp((turns - BETA_SLOW) / (BETA_FAST - BETA_SLOW), 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / case["factor"])
    return f


def _rotate(x, cos, sin, case):
    """x [b, s, heads, dim], cos / sin [b, s, 1, pairs]; x's own type but for the rotation's."""
    rot = case["rot_dim"]
    head, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "interleaved":
        a, b = head[..., 0::2], head[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y, rest), dim=-1)


def _rope_heads(x, kept, cos, sin, case, most, dtype):
    """The first `most` heads rotated, rows past the lengths zero."""
    y = torch.cat((_rotate(x[:, :, :most], cos, sin, case), x[:, :, most:]), dim=2)
    return (y if kept is None else torch.where(kept, y, torch.zeros((), dtype=y.dtype, device=DEV))).to(dtype)


def _rope_outputs(st, work_type):
    case = st["case"]
    b, s = case["batch"], case["seq"]
    pos = torch.arange(s, device=DEV).expand(b, s) if st["positions"] is None else st["positions"]
    angle = pos.double()[:, :, None, None] * _frequencies(case)
    cos, sin = torch.cos(angle).to(work_type), torch.sin(angle).to(work_type)
    if case["inverse"]:
        sin = -sin
    kept = None
    if st["lengths"] is not None:
        kept = (torch.arange(s, device=DEV)[None] < st["lengths"][:, None])[:, :, None, None]
    out = work_type if work_type == torch.float64 else TYPE[case["dtype"]]
    return {"q": _rope_heads(st["q"].to(work_type), kept, cos, sin, case, case["rot_heads"], out),
            "k": _rope_heads(st["k"].to(work_type), kept, cos, sin, case, min(case["rot_heads"], case["kv_heads"]), out)}


def _plain_cross(st):
    case = st["case"]
    b, sq, skv, h, hk, d = (case[x] for x in ("batch", "sq", "skv", "heads", "kv_heads", "dim"))
    q = st["q"].float().reshape(b, sq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * sq, d)
    kt = st["k"].float().permute(0, 2, 3, 1).contiguous()
    v = st["v"].float().permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q, kt) * d ** -0.5
    on = None
    if st["lengths"] is not None:
        on = torch.arange(skv, device=DEV)[None] < st["lengths"][:, None]
    if st["mask"] is not None:
        on = st["mask"] != 0 if on is None else on & (st["mask"] != 0)
    if on is not None:
        scores = scores.masked_fill(~on[:, None, None, :], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(b, hk, h // hk, sq, d).permute(0, 3, 1, 2, 4).reshape(b, sq, h, d)
    return {"out": o.to(TYPE[case["dtype"]])}


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
    """What a program makes once per shape: the call's description and its workspace."""
    if st["plan"] is None:
        ih, case = _package(), st["case"]
        if case["kind"] == "linear":
            desc = ih.LinearDesc(case["m"], case["n"], case["k"], dtype=case["dtype"], out_dtype=case["out"],
                                 activation=case["act"], gate_rows=case["gate_rows"])
            nbytes = ih.ops.linear_workspace(desc)
        elif case["kind"] == "rope":
            desc = ih.RopeDesc(case["batch"], case["seq"], case["dim"], heads=case["heads"], kv_heads=case["kv_heads"],
                               dtype=case["dtype"], layout=case["layout"], rot_dim=case["rot_dim"], rot_heads=case["rot_heads"],
                               rot_kv_heads=min(case["rot_heads"], case["kv_heads"]), theta=case["theta"],
                               scaling=case["scaling"], factor=case["factor"], trained_len=TRAINED, beta_fast=BETA_FAST,
                               beta_slow=BETA_SLOW, inverse=case["inverse"], q_strides=st["q"].stride()[:3],
                               k_strides=st["k"].stride()[:3])
            nbytes = 0
        else:
            desc = ih.CrossAttentionDesc(case["batch"], case["sq"], case["skv"], case["heads"], case["kv_heads"], case["dim"],
                                         dtype=case["dtype"], k_strides=st["k"].stride()[:3], v_strides=st["v"].stride()[:3])
            nbytes = ih.ops.cross_attention_workspace(desc)
        st["plan"] = (ih.ops, desc, torch.empty(nbytes, dtype=torch.uint8, device=DEV) if nbytes else None, nbytes)
    return st["plan"]


def _own(st):
    ops, desc, ws, nbytes = _plan(st)
    kind, stream = st["case"]["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "linear":
        ops.linear(desc, _ptr(st["x"]), _ptr(st["w"]), _ptr(st["y"]), d_bias=_ptr(st["bias"]), d_gate=_ptr(st["gate"]),
                   d_residual=_ptr(st["residual"]), d_workspace=_ptr(ws), workspace_bytes=nbytes, stream=stream)
        return {"y": st["y"]}
    if kind == "rope":
        ops.rope(desc, _ptr(st["q"]), _ptr(st["q_out"]), _ptr(st["k"]), _ptr(st["k_out"]), d_positions=_ptr(st["positions"]),
                 d_lengths=_ptr(st["lengths"]), stream=stream)
        return {"q": st["q_out"], "k": st["k_out"]}
    ops.cross_attention(desc, _ptr(st["q"]), _ptr(st["k"]), _ptr(st["v"]), _ptr(st["out"]), d_mask=_ptr(st["mask"]),
                        d_kv_len=_ptr(st["lengths"]), d_workspace=_ptr(ws), workspace_bytes=nbytes, stream=stream)
    return {"out": st["out"]}


def run(st):
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    if kind == "linear":
        return _plain_linear(st)
    if kind == "rope":
        return _rope_outputs(st, torch.float32)
    return _plain_cross(st)


# ---- the work, and the outputs in float64 -------------------------------------------------------
def work(case):
    es = SIZE[case["dtype"]]
    if case["kind"] == "linear":
        m, n, k, eo = case["m"], case["n"], case["k"], SIZE[case["out"]]
        nbytes = (m * k + n * k) * es + m * n * eo * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0)
        if case["gate_rows"]:
            nbytes += 4 * n * -(-m // case["gate_rows"])
        return {"bytes": nbytes, "flops": 2 * m * n * k}
    if case["kind"] == "rope":
        rows = sum(_lengths(case["batch"], case["seq"])) if case["ragged"] else case["batch"] * case["seq"]
        heads = case["heads"] + case["kv_heads"]
        turned = case["rot_heads"] + min(case["rot_heads"], case["kv_heads"])
        return {"bytes": 2 * rows * heads * case["dim"] * es + (4 * rows if case["far"] else 0),
                "flops": 3 * rows * turned * case["rot_dim"]}
    b, sq, skv, h, hk, d = (case[x] for x in ("batch", "sq", "skv", "heads", "kv_heads", "dim"))
    lens = _lengths(b, skv) if case["ragged"] else [skv] * b
    if case["masked"]:
        lens = [n * 0.9 for n in lens]
        if b > 1:
            lens[-1] = 0  # the dropped condition
    keys = sum(lens)
    return {"bytes": int(2 * b * sq * h * d * es + 2 * keys * hk * d * es + (b * skv if case["masked"] else 0)),
            "flops": int(4 * keys * sq * h * d)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "linear":
        y = st["x"].double() @ st["w"].double().T
        if st["bias"] is not None:
            y += st["bias"].double()
        y = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
             "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]](y)
        if st["gate"] is not None:
            y *= st["gate"].double()[torch.arange(case["m"], device=DEV) // case["gate_rows"]]
        if st["residual"] is not None:
            y += st["residual"].double()
        return {"y": y}
    if case["kind"] == "rope":
        # As complex numbers: a pair is multiplied by exp(i angle).
        b, s, rot = case["batch"], case["seq"], case["rot_dim"]
        factor, theta = case["factor"], case["theta"]
        freq = []
        for i in range(rot // 2):
            if case["scaling"] == "ntk":
                freq.append((theta * factor ** (rot / (rot - 2))) ** (-2 * i / rot))
                continue
            f = theta ** (-2 * i / rot)
            if case["scaling"] == "linear":
                f /= factor
            elif case["scaling"] == "by_parts":
                share = min(1.0, max(0.0, (TRAINED * f / math.tau - BETA_SLOW) / (BETA_FAST - BETA_SLOW)))
                f = share * f + (1.0 - share) * f / factor
            freq.append(f)
        pos = torch.arange(s, device=DEV).repeat(b, 1) if st["positions"] is None else st["positions"]
        angle = pos.double().unsqueeze(-1) * torch.tensor(freq, dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle).unsqueeze(2)
        res = {}
        for name, most in (("q", case["rot_heads"]), ("k", min(case["rot_heads"], case["kv_heads"]))):
            y = st[name].double().clone()
            part = y[:, :, :most, :rot]
            if case["layout"] == "interleaved":
                z = torch.view_as_complex(part.reshape(b, s, most, rot // 2, 2).contiguous()) * turn
                y[:, :, :most, :rot] = torch.view_as_real(z).reshape(b, s, most, rot)
            else:
                z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * turn
                y[:, :, :most, :rot] = torch.cat([z.real, z.imag], -1)
            if st["lengths"] is not None:
                for row, n in enumerate(st["lengths"].tolist()):
                    y[row, n:] = 0
            res[name] = y
        return res
    b, sq, skv, h, hk, d = (case[x] for x in ("batch", "sq", "skv", "heads", "kv_heads", "dim"))
    out = torch.zeros(b, sq, h, d, dtype=torch.float64, device=DEV)
    for row in range(b):
        keys = torch.arange(skv, device=DEV)
        if st["lengths"] is not None:
            keys = keys[:int(st["lengths"][row])]
        if st["mask"] is not None:
            keys = keys[st["mask"][row, keys] != 0]
        if keys.numel() == 0:
            continue
        for head in range(h):
            kk, vv = st["k"][row, keys, head // (h // hk)].double(), st["v"][row, keys, head // (h // hk)].double()
            weights = torch.softmax(st["q"][row, :, head].double() @ kk.T / math.sqrt(d), dim=-1)
            out[row, :, head] = weights @ vv
    return {"out": out}
