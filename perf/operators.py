"""What the expert-MLP operators in 4-bit floating point and in 16 bits are measured on.

A case is one call (or the calls that belong to one layer) of

  quantise    ``quantize_fp4`` and ``dequantize_fp4``: rows to e2m1 with block scales, and the values they stand for
  product     ``grouped_gemm_fp4``: the rows of every expert times that expert's 4-bit weights
  fp4_mlp     ``quantize_fp4`` -> ``grouped_gemm_fp4_swiglu`` -> ``grouped_gemm_fp4``: a 4-bit expert MLP
  mlp         ``grouped_mlp``: the gated feed-forward block of unquantised experts
  mlp_train   the same with its backward pass: gradients of the rows and of both weights

Formats: ``nvfp4`` has one e4m3 scale per 16 values and a fp32 scale per tensor (rows) or per expert (weights); ``mxfp4`` has
one power-of-two scale (e8m0) per 32 values.  Rows are grouped by expert: expert e owns rows offsets[e] .. offsets[e + 1].
Rows past offsets[-1] (the padding of a receive buffer) belong to no expert; their outputs and gradients are zero.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False  # True: run() makes the library's calls, False: elementary torch operations in fp32

DEV = "cuda"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def _case(name, op, rows, hidden, inter=0, experts=1, idle=0, skew=0.0, fmt="", dtype="bf16", pad=0):
    c = dict(op=op, rows=rows, hidden=hidden, inter=inter, experts=experts, idle=idle, skew=skew, fmt=fmt, dtype=dtype, pad=pad)
    return dict(c, name=name) if name else c


def listed():
    return [
        # rows of a decode batch before the first product
        _case("quantise decode", "quantise", 128, 7168, fmt="nvfp4"),
        # rows of a prefill batch after dispatch
        _case("quantise prefill", "quantise", 32768, 7168, fmt="nvfp4"),
        # a few experts' weights moved to 4 bits when a checkpoint is loaded
        _case("quantise weights mx", "quantise", 24576, 4096, fmt="mxfp4", dtype="fp32"),
        # down projection of one rank's 32 experts in decode: 128 tokens of each of 8 ranks, uneven experts
        _case("product decode", "product", 1024, 2048, 7168, experts=32, idle=3, skew=0.5, fmt="nvfp4"),
        # the same weights in prefill: 4096 tokens per rank
        _case("product prefill", "product", 32768, 2048, 7168, experts=32, skew=0.2, fmt="nvfp4"),
        # one token whose eight experts all live on this rank
        _case("fp4 mlp one token", "fp4_mlp", 8, 7168, 2048, experts=32, idle=24, fmt="nvfp4"),
        # a decode layer of mxfp4 experts, buffer larger than the rows received
        _case("fp4 mlp decode mx", "fp4_mlp", 600, 4096, 1024, experts=32, idle=2, skew=0.7, fmt="mxfp4", pad=168),
        # a prefill layer
        _case("fp4 mlp prefill", "fp4_mlp", 16384, 7168, 2048, experts=16, skew=0.2, fmt="nvfp4"),
        # the shared (unquantised) expert of a layer on a single token
        _case("shared expert one token", "mlp", 1, 7168, 2048),
        # unquantised experts in a prefill step, uneven experts, fp16 checkpoint
        _case("mlp prefill", "mlp", 9001, 4096, 1024, experts=24, idle=1, skew=0.6, dtype="fp16", pad=215),
        # fine-tuning of small experts with odd sizes
        _case("train small", "mlp_train", 777, 1000, 344, experts=6, idle=1, skew=0.5),
        # a training step of one rank's experts
        _case("train step", "mlp_train", 16384, 4096, 2048, experts=16, skew=0.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["quantise", "product", "fp4_mlp", "mlp", "mlp_train"])
        fmt = rng.choice(["nvfp4", "mxfp4"])
        if op == "quantise":
            return _case("", op, _log(rng, 1, 32768), 32 * rng.randint(2, 224), fmt=fmt, dtype=rng.choice(["bf16", "fp16", "fp32"][: 2 if rng.random() < 0.7 else 3]))
        step = 8 if op.startswith("mlp") else 128
        hidden = step * rng.randint(512 // step, 7168 // step)
        inter = step * rng.randint(max(1, 256 // step), 2048 // step)
        if op == "product" and rng.random() < 0.5:
            hidden, inter = inter, hidden
        experts = _log(rng, 1, 32)
        rows = _log(rng, 1, 32768)
        idle = rng.randint(0, experts // 3)
        c = _case("", op, rows, hidden, inter, experts=experts, idle=idle, skew=round(rng.uniform(0.0, 0.9), 2), fmt=fmt if "mlp" != op[:3] else "",
                  dtype="bf16" if "fp4" in op or op == "product" else rng.choice(["bf16", "fp16"]), pad=rng.choice([0, 0, rng.randint(1, 300)]))
        most = {"product": 1.0e12, "fp4_mlp": 1.5e12, "mlp": 9e11, "mlp_train": 1.8e12}[op]
        weights = {"mlp": 16 * 7168 * 2048, "mlp_train": 16 * 4096 * 2048}.get(op, 32 * 7168 * 2048)
        if work(c)["flops"] <= most and experts * hidden * inter <= weights:
            return c


def _live(c):
    return max(1, min(c["experts"] - c["idle"], c["rows"]))


def work(c):
    m, h, i, live = c["rows"], c["hidden"], c["inter"], _live(c)
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
    q = 0.5 + (1 / 16 if c["fmt"] == "nvfp4" else 1 / 32)  # bytes of a 4-bit value with its share of the scale
    if c["op"] == "quantise":
        n = m * h
        # rows in, codes and scales out; the values come back as bf16 from the codes and scales
        return {"bytes": n * size + 2 * n * q + 2 * n, "flops": 4 * n}
    if c["op"] == "product":
        return {"bytes": m * h * q + live * h * i * q + m * i * 2, "flops": 2 * m * h * i}
    if c["op"] == "fp4_mlp":
        return {"bytes": 2 * m * h * 2 + live * 3 * h * i * q, "flops": 2 * m * 3 * h * i}
    if c["op"] == "mlp":
        return {"bytes": 2 * m * h * 2 + live * 3 * h * i * 2, "flops": 2 * m * 3 * h * i}
    # x, dy, y, dx and the weights once, every expert's weight gradients once
    return {"bytes": 4 * m * h * 2 + (live + c["experts"]) * 3 * h * i * 2, "flops": 3 * 2 * m * 3 * h * i}


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _counts(c, seed):
    """Rows of every expert: `_live` of them get one row at least, the rest is shared out unevenly."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    live, rows, e = _live(c), c["rows"], c["experts"]
    at = torch.randperm(e, generator=g)[:live]
    share = torch.exp(torch.randn(live, generator=g) * c["skew"]).double()
    extra = torch.floor(share / share.sum() * (rows - live)).long()
    extra[0] += rows - live - int(extra.sum())
    counts = torch.zeros(e, dtype=torch.long)
    counts[at] = extra + 1
    return counts


def _fp4_weights(shape, fmt, std, g):
    """N(0, std) weights in 4 bits: codes of the bell curve, block scales that vary a little, one fp32 scale per expert."""
    e, n, k = shape
    block = 16 if fmt == "nvfp4" else 32
    q = torch.empty(e, n, k // 2, dtype=torch.uint8, device=DEV)
    for j in range(e):
        v = torch.randn(n, k, device=DEV, generator=g, dtype=torch.float16) * 2.9
        code = torch.bucketize(v.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV, dtype=torch.float16), out_int32=True).to(torch.uint8)
        code |= (v < 0).to(torch.uint8) << 3
        q[j] = code[:, 0::2] | (code[:, 1::2] << 4)
    u = torch.rand(e, n, k // block, device=DEV, generator=g)
    if fmt == "nvfp4":
        s = (64.0 * (0.7 + 0.6 * u)).to(torch.float8_e4m3fn)
        gs = std / 2.9 / 64.0 * (0.9 + 0.2 * torch.rand(e, device=DEV, generator=g))
        return q, s, gs
    top = round(math.log2(std / 2.9))
    s = (top + 127 + torch.floor(2 * u) - 1).to(torch.uint8).view(torch.float8_e8m0fnu)
    return q, s, None


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    m, h, i, e = c["rows"] + c["pad"], c["hidden"], c["inter"], c["experts"]
    dt = DTYPES[c["dtype"]]
    s = {"case": {k: v for k, v in c.items() if k != "name"}, "block": 16 if c["fmt"] == "nvfp4" else 32}
    if c["op"] == "quantise":
        # activations have channels of very different size
        x = torch.randn(m, h, device=DEV, generator=g) * torch.exp(torch.randn(h, device=DEV, generator=g))
        s["x"] = x.to(dt)
        s["x_gs"] = torch.full((1,), 1.0 / 128, device=DEV) if c["fmt"] == "nvfp4" else None
        return s
    counts = _counts(c, seed)
    off = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    s["offsets"] = off.to(torch.int32).to(DEV)
    s["cap"] = int(counts.max())
    # place of every row in a [experts, cap] array: the plan of the padded products of the plain form
    owner = torch.repeat_interleave(torch.arange(e), counts)
    s["slots"] = (owner * s["cap"] + torch.arange(c["rows"]) - off[owner]).to(DEV)
    x = torch.randn(m, h, device=DEV, generator=g)
    nv = c["fmt"] == "nvfp4"
    if c["op"] == "product":
        # rows as a quantised SwiGLU output leaves them
        block = s["block"]
        code = torch.bucketize((x * 2.4).abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)).to(torch.uint8)
        code |= (x < 0).to(torch.uint8) << 3
        s["a_q"] = code[:, 0::2] | (code[:, 1::2] << 4)
        u = torch.rand(m, h // block, device=DEV, generator=g)
        s["a_s"] = (32.0 * (0.25 + u)).to(torch.float8_e4m3fn) if nv else (125 + torch.floor(3 * u)).to(torch.uint8).view(torch.float8_e8m0fnu)
        s["a_gs"] = torch.full((1,), 1.0 / 64, device=DEV) if nv else None
        s["w_q"], s["w_s"], s["w_gs"] = _fp4_weights((e, i, h), c["fmt"], h ** -0.5, g)
        return s
    if c["op"] == "fp4_mlp":
        s["x"] = x.to(dt)
        s["x_gs"] = torch.full((1,), 1.0 / 256, device=DEV) if nv else None
        s["act_gs"] = torch.full((1,), 1.0 / 100, device=DEV) if nv else None
        s["w1_q"], s["w1_s"], s["w1_gs"] = _fp4_weights((e, 2 * i, h), c["fmt"], h ** -0.5, g)
        s["w2_q"], s["w2_s"], s["w2_gs"] = _fp4_weights((e, h, i), c["fmt"], i ** -0.5, g)
        return s
    train = c["op"] == "mlp_train"
    s["x"] = x.to(dt).requires_grad_(train)
    s["w1"] = (torch.randn(e, 2 * i, h, device=DEV, generator=g, dtype=dt) * h ** -0.5).requires_grad_(train)
    s["w2"] = (torch.randn(e, h, i, device=DEV, generator=g, dtype=dt) * i ** -0.5).requires_grad_(train)
    if train:
        s["dy"] = torch.randn(m, h, device=DEV, generator=g, dtype=dt)
    return s


# ------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------
def _quantise(x, block, gs):
    """fp32 values -> (e2m1 values, scales as fp32): s = e4m3(amax / (6 gs)), or the smallest power of two >= amax / 6."""
    v = x.reshape(*x.shape[:-1], -1, block)
    amax = v.abs().amax(-1)
    if gs is not None:
        s = (amax / (6.0 * gs)).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        d = s * gs
    else:
        m, ex = torch.frexp(amax / 6.0)
        code = (ex + 127 - (m == 0.5).int()).clamp(1, 254) * (amax > 0)
        s = torch.exp2((code - 127).double()).float()
        d = s
    y = torch.where(d[..., None] > 0, v / d[..., None], torch.zeros_like(v))
    a = y.abs()
    step = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).long()
    val = torch.tensor(E2M1, device=x.device)[step]
    return torch.where(y < 0, -val, val), s


def _values(q, s, gs, block):
    """Packed codes and scales -> fp32 values."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
    v = torch.stack([table[(q & 15).int()], table[(q >> 4).int()]], -1).flatten(-2)
    d = s.float() if s.dtype == torch.float8_e4m3fn else torch.exp2((s.view(torch.uint8).int() - 127).double()).float()
    if gs is not None:
        d = d * gs.reshape(-1, *([1] * (d.dim() - 1)))
    return v * d.repeat_interleave(block, -1)


def _padded(x, st):
    c = st["case"]
    out = x.new_zeros(c["experts"] * st["cap"], x.shape[1])
    out[st["slots"]] = x[: c["rows"]]
    return out.view(c["experts"], st["cap"], -1)


def _rows(y, st):
    c = st["case"]
    return torch.cat([y.reshape(-1, y.shape[-1])[st["slots"]], y.new_zeros(c["pad"], y.shape[-1])])


def _swiglu(gu):
    g, u = gu.chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def _run_plain(st):
    c, block = st["case"], st["block"]
    if c["op"] == "quantise":
        val, s = _quantise(st["x"].float(), block, st["x_gs"])
        d = s if st["x_gs"] is None else s * st["x_gs"]
        return {"values": (val * d[..., None]).flatten(-2).to(torch.bfloat16), "scales": s.to(torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu)}
    if c["op"] == "product":
        a = _padded(_values(st["a_q"], st["a_s"], st["a_gs"], block), st)
        w = _values(st["w_q"], st["w_s"], st["w_gs"], block)
        return _rows(torch.bmm(a, w.transpose(1, 2)), st).to(torch.bfloat16)
    if c["op"] == "fp4_mlp":
        val, s = _quantise(st["x"].float(), block, st["x_gs"])
        d = s if st["x_gs"] is None else s * st["x_gs"]
        x = _padded((val * d[..., None]).flatten(-2), st)
        act = _swiglu(torch.bmm(x, _values(st["w1_q"], st["w1_s"], st["w1_gs"], block).transpose(1, 2)))
        val, s = _quantise(act, block, st["act_gs"])
        d = s if st["act_gs"] is None else s * st["act_gs"]
        act = (val * d[..., None]).flatten(-2)
        return _rows(torch.bmm(act, _values(st["w2_q"], st["w2_s"], st["w2_gs"], block).transpose(1, 2)), st).to(torch.bfloat16)
    dt = st["x"].dtype
    x, w1, w2 = _padded(st["x"].detach().float(), st), st["w1"].detach().float(), st["w2"].detach().float()
    gu = torch.bmm(x, w1.transpose(1, 2))
    act = _swiglu(gu)
    y = _rows(torch.bmm(act, w2.transpose(1, 2)), st).to(dt)
    if c["op"] == "mlp":
        return y
    dy = _padded(st["dy"].float(), st)
    dact = torch.bmm(dy, w2)
    dw2 = torch.bmm(dy.transpose(1, 2), act)
    g, u = gu.chunk(2, -1)
    sig = 1 / (1 + torch.exp(-g))
    dgu = torch.cat([dact * u * sig * (1 + g * (1 - sig)), dact * g * sig], -1)
    return {"y": y, "dx": _rows(torch.bmm(dgu, w1), st).to(dt), "dw1": torch.bmm(dgu.transpose(1, 2), x).to(dt), "dw2": dw2.to(dt)}


# ------------------------------------------------------------------------------------------------
# The library's calls
# ------------------------------------------------------------------------------------------------
def _run_own(st):
    from umdk_original_b200 import ops
    c, block = st["case"], st["block"]
    if c["op"] == "quantise":
        q, s = ops.quantize_fp4(st["x"], block, st["x_gs"])
        return {"values": ops.dequantize_fp4(q, s, st["x_gs"]), "scales": s}
    if c["op"] == "product":
        return ops.grouped_gemm_fp4(st["a_q"], st["a_s"], st["w_q"], st["w_s"], st["offsets"], st["a_gs"], st["w_gs"])
    if c["op"] == "fp4_mlp":
        q, s = ops.quantize_fp4(st["x"], block, st["x_gs"])
        q, s = ops.grouped_gemm_fp4_swiglu(q, s, st["w1_q"], st["w1_s"], st["offsets"], st["x_gs"], st["w1_gs"], st["act_gs"])
        return ops.grouped_gemm_fp4(q, s, st["w2_q"], st["w2_s"], st["offsets"], st["act_gs"], st["w2_gs"])
    y = ops.grouped_mlp(st["x"], st["w1"], st["w2"], st["offsets"])
    if c["op"] == "mlp":
        return y
    dx, dw1, dw2 = torch.autograd.grad(y, (st["x"], st["w1"], st["w2"]), st["dy"])
    return {"y": y, "dx": dx, "dw1": dw1, "dw2": dw2}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits, expert by expert
# ------------------------------------------------------------------------------------------------
def _exact_scale_product(x, nv, gs):
    """(x rounded to 4 bits with its block scales, the scales), in fp64."""
    b = 16 if nv else 32
    v = x.double().unflatten(-1, (-1, b))
    top = v.abs().max(-1).values / 6
    if nv:
        t = (top / gs).clamp(max=448)
        e = torch.floor(torch.log2(t.clamp(min=2.0 ** -6)))
        ulp = torch.exp2(e - 3)  # e4m3: three bits behind the point, exponents from -6
        s = torch.round(t / ulp) * ulp
        d = s * gs
    else:
        s = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -126))))
        s = torch.where(top > 0, s, torch.full_like(s, 2.0 ** -127))
        d = s
    r = v / torch.where(d > 0, d, torch.ones_like(d))[..., None]
    a = r.abs()
    unit = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    n = (torch.round(a / unit) * unit).clamp(max=6) * torch.sign(r)
    return torch.where(d[..., None] > 0, n * d[..., None], torch.zeros_like(n)).flatten(-2), s


def _exact_values(q, s, gs):
    lo, hi = (q & 15).long(), (q >> 4).long()
    c = torch.stack((lo, hi), -1).flatten(-2)
    ex, mant = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(ex == 0, mant / 2, torch.exp2((ex - 1).double()) * (1 + mant / 2))
    v = torch.where(c >= 8, -mag, mag)
    n = v.shape[-1] // s.shape[-1]
    d = s.double() if s.dtype == torch.float8_e4m3fn else torch.exp2(s.view(torch.uint8).double() - 127)
    return (v.unflatten(-1, (-1, n)) * d[..., None]).flatten(-2) * (1.0 if gs is None else gs.double())


def exact(c, seed):
    st = prepare(c, seed)
    nv = c["fmt"] == "nvfp4"
    if c["op"] == "quantise":
        if c["rows"] * c["hidden"] > 120_000_000:
            parts = [_exact_scale_product(p, nv, st["x_gs"].double() if nv else None) for p in st["x"].split(4096)]
            return {"values": torch.cat([p[0].float() for p in parts]).double(), "scales": torch.cat([p[1] for p in parts])}
        v, s = _exact_scale_product(st["x"], nv, st["x_gs"].double() if nv else None)
        return {"values": v, "scales": s}
    off = st["offsets"].tolist()
    m, e = c["rows"] + c["pad"], c["experts"]
    silu = lambda g: g * torch.sigmoid(g)  # noqa: E731
    gs = lambda k, j: None if st[k] is None else st[k][j: j + 1]  # noqa: E731
    if c["op"] in ("product", "fp4_mlp"):
        n = c["inter"] if c["op"] == "product" else c["hidden"]
        y = torch.zeros(m, n, device=DEV, dtype=torch.float64)
        for j in range(e):
            a, b = off[j], off[j + 1]
            if a == b:
                continue
            if c["op"] == "product":
                rows = _exact_values(st["a_q"][a:b], st["a_s"][a:b], st["a_gs"])
                y[a:b] = rows @ _exact_values(st["w_q"][j], st["w_s"][j], gs("w_gs", j)).T
            else:
                rows, _ = _exact_scale_product(st["x"][a:b], nv, st["x_gs"].double() if nv else None)
                gate, up = (rows @ _exact_values(st["w1_q"][j], st["w1_s"][j], gs("w1_gs", j)).T).chunk(2, -1)
                rows, _ = _exact_scale_product(silu(gate) * up, nv, st["act_gs"].double() if nv else None)
                y[a:b] = rows @ _exact_values(st["w2_q"][j], st["w2_s"][j], gs("w2_gs", j)).T
        return y
    out = {"y": torch.zeros(m, c["hidden"], device=DEV, dtype=torch.float64)}
    train = c["op"] == "mlp_train"
    if train:
        out |= {"dx": torch.zeros_like(out["y"]), "dw1": torch.zeros(st["w1"].shape, device=DEV, dtype=torch.float64),
                "dw2": torch.zeros(st["w2"].shape, device=DEV, dtype=torch.float64)}
    for j in range(e):
        a, b = off[j], off[j + 1]
        if a == b:
            continue
        # the derivative of the written-down formula by reverse mode in fp64, not by the plain form's expressions
        x, w1, w2 = (t.detach().double().requires_grad_(train) for t in (st["x"][a:b], st["w1"][j], st["w2"][j]))
        gate, up = F.linear(x, w1).chunk(2, -1)
        y = F.linear(silu(gate) * up, w2)
        out["y"][a:b] = y.detach()
        if train:
            out["dx"][a:b], out["dw1"][j], out["dw2"][j] = torch.autograd.grad(y, (x, w1, w2), st["dy"][a:b].double())
    return out if train else out["y"]
