"""What the operators around the experts are measured on: norm, routing, rows to the experts and back.

A case is one call (or the calls that belong together) of

  norm          ``add_rms_norm``: the residual's addition and the root-mean-square norm of the sum
  norm_train    the same with its backward pass
  norm_quant    ``rms_norm_quant``: the same with the normalised rows in 8 bits (quant modes of the dispatch: 2 int8 with a scale
                per row, 3 e4m3 with fp32 scales per 128 values, 4 e4m3 with power-of-two scales)
  route         ``moe_route``: experts and weights of every token from its logits
  route_train   the same with its backward pass
  regroup       ``moe_group_rows`` and ``moe_ungroup_rows``: rows sorted by expert, and the experts' results brought back
  regroup_train the same with the backward passes of both

The sum of a residual's addition is rounded to the residual's type, and the norm is that of the rounded sum.  Rows of one expert keep
the order of their (token, choice) pairs; pairs whose id is negative (tokens of padding) belong to no expert, and the rows that are
left at the end are zeros.
"""
from __future__ import annotations

import math

import torch

own = False  # True: run() makes the library's calls, False: elementary torch operations

DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def _case(name, op, tokens, hidden=0, dtype="bf16", residual="same", mode=0, experts=0, topk=0, groups=1, topk_groups=1, score="softmax",
          bias=False, renorm=True, skew=0.0, idle=0.0):
    c = dict(op=op, tokens=tokens, hidden=hidden, dtype=dtype, residual=residual, mode=mode, experts=experts, topk=topk, groups=groups,
             topk_groups=topk_groups, score=score, bias=bias, renorm=renorm, skew=skew, idle=idle)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a small decode batch before a layer
        _case("norm decode", "norm", 61, 7168),
        # a prefill batch, fp32 residual stream
        _case("norm prefill", "norm", 16384, 4096, residual="fp32"),
        # a training step of one rank
        _case("norm train", "norm_train", 8192, 7168),
        # decode rows that go to 8-bit experts
        _case("norm quant decode", "norm_quant", 128, 7168, mode=3),
        # prefill rows of a W8A8 layer go out with e4m3 and power-of-two scales
        _case("norm quant prefill", "norm_quant", 32768, 7168, mode=4),
        # decode routing, sigmoid scores with a selection bias, 4 of 8 groups
        _case("route decode", "route", 128, experts=256, topk=8, groups=8, topk_groups=4, score="sigmoid", bias=True, dtype="fp32"),
        # prefill routing, plain softmax over 128 experts
        _case("route prefill", "route", 32768, experts=128, topk=8),
        # routing of a training step with its gradient
        _case("route train", "route_train", 16384, experts=256, topk=8, groups=8, topk_groups=4, score="sigmoid", bias=True, dtype="fp32"),
        # one decode batch of 8-bit rows with their scales, a few tokens of padding
        _case("regroup decode 8 bit", "regroup", 128, 7168, dtype="e4m3", experts=256, topk=8, skew=0.5, idle=0.05),
        # prefill, 16-bit rows
        _case("regroup prefill", "regroup", 4096, 7168, experts=256, topk=8, skew=0.3),
        # fine-tuning on few tokens of an odd width
        _case("regroup train small", "regroup_train", 777, 1000, dtype="fp16", experts=6, topk=2, skew=0.5, idle=0.1),
        # a training step
        _case("regroup train", "regroup_train", 8192, 4096, experts=128, topk=8, skew=0.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["norm", "norm_train", "norm_quant", "route", "route_train", "regroup", "regroup_train"])
        tokens = _log(rng, 1, 32768)
        step = rng.choice([128, 128, 8, 1])
        hidden = step * _log(rng, max(1, 64 // step), 8192 // step)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if op.startswith("norm"):
            mode = rng.choice([2, 3, 4]) if op == "norm_quant" else 0
            c = _case("", op, tokens, 128 * max(1, hidden // 128) if mode > 2 else hidden, dtype=dtype,
                      residual=rng.choice(["same", "same", "fp32", "none"][: 4 if op == "norm_quant" else 3]), mode=mode)
        else:
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = groups * max(2, _log(rng, 4, 384) // groups)
            topk_groups = rng.randint(1, groups)
            k = rng.randint(2, min(10, experts // groups * topk_groups))  # one weight alone, renormalised, is 1 and has no gradient
            if op.startswith("route"):
                score = rng.choice(["softmax", "sigmoid"])
                c = _case("", op, tokens, dtype=dtype, experts=experts, topk=k, groups=groups, topk_groups=topk_groups, score=score,
                          bias=rng.random() < 0.5, renorm=rng.random() < 0.7)
            else:
                if op == "regroup" and rng.random() < 0.3:
                    dtype, hidden = "e4m3", 128 * max(1, hidden // 128)
                c = _case("", op, tokens, hidden, dtype=dtype, experts=experts, topk=k, skew=round(rng.uniform(0.0, 0.9), 2),
                          idle=rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.3), 2)]))
        if work(c)["bytes"] <= top:
            return c


def _res_size(c):
    return {"same": SIZES[c["dtype"]], "fp32": 4, "none": 0}[c["residual"]]


def work(c):
    t, h, e, k = c["tokens"], c["hidden"], c["experts"], c["topk"]
    b = SIZES[c["dtype"]]
    if c["op"].startswith("norm"):
        r = _res_size(c)
        n = t * h
        if c["op"] == "norm":
            return {"bytes": n * (2 * b + 2 * r) + h * b, "flops": 5 * n}
        if c["op"] == "norm_quant":
            scales = t * 4 if c["mode"] == 2 else t * (h // 128) * 4
            return {"bytes": n * (b + 2 * r + 1) + scales + h * b, "flops": 7 * n}
        # x, r, dy, ds in; y, s, the gradients of x and (of another type) r out
        return {"bytes": n * (2 * b + 2 * r + b + r + (0 if c["dtype"] == "fp32" or c["residual"] == "same" else r)) + 2 * h * b, "flops": 15 * n}
    if c["op"].startswith("route"):
        n = t * e
        fwd = {"bytes": n * b + t * k * 12 + (e * 4 if c["bias"] else 0), "flops": 6 * n + 4 * t * k}
        if c["op"] == "route":
            return fwd
        return {"bytes": fwd["bytes"] + t * k * 4 + n * b, "flops": fwd["flops"] + 2 * n}
    pairs = t * k
    b_out = 2 if c["dtype"] == "e4m3" else b
    small = pairs * (8 + 4 + 4) + (e + 1) * 4 + ((t + pairs) * (h // 128) * 4 if c["dtype"] == "e4m3" else 0)
    live = int(round(pairs * (1 - c["idle"])))
    fwd = {"bytes": (t + pairs) * h * b + (live + t) * h * b_out + small, "flops": 2 * live * h}
    if c["op"] == "regroup":
        return fwd
    # gradients of rows and output in; gradients of x, of the experts' results and of the weights out
    return {"bytes": fwd["bytes"] + (live + t) * h * b + (t + pairs) * h * b + pairs * 4, "flops": 6 * live * h}


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g, dtype=torch.float32 if dtype == torch.float8_e4m3fn else dtype).to(dtype)


def _routing(c, g):
    """Distinct expert ids per token, uneven over the experts; tokens of padding have -1."""
    t, e, k = c["tokens"], c["experts"], c["topk"]
    z = torch.randn(e, device=DEV, generator=g) * c["skew"] * 2
    u = torch.rand(t, e, device=DEV, generator=g).clamp_(1e-9, 1.0)
    idx = torch.topk(z - torch.log(-torch.log(u)), k, dim=-1).indices
    w = torch.softmax(torch.randn(t, k, device=DEV, generator=g), -1)
    if c["idle"]:
        idx = torch.where(torch.rand(t, 1, device=DEV, generator=g) < c["idle"], torch.full_like(idx, -1), idx)
    return idx, w


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, h, dt = c["tokens"], c["hidden"], DTYPES[c["dtype"]]
    s = {"case": {k: v for k, v in c.items() if k != "name"}}
    train = c["op"].endswith("train")
    if c["op"].startswith("norm"):
        rdt = {"same": dt, "fp32": torch.float32, "none": None}[c["residual"]]
        channels = torch.exp(0.5 * torch.randn(h, device=DEV, generator=g))  # channels of different size
        s["x"] = (_randn(g, t, h) * channels).to(dt)
        s["residual"] = None if rdt is None else (2 * _randn(g, t, h) * channels).to(rdt)
        s["weight"] = (1 + 0.2 * _randn(g, h)).to(dt)
        if train:
            s["dy"], s["dsum"] = _randn(g, t, h, dtype=dt), _randn(g, t, h, dtype=rdt)
            for name in ("x", "residual", "weight"):
                s[name].requires_grad_()
        return s
    if c["op"].startswith("route"):
        # logits of a trained gate: some experts are liked more than others
        s["logits"] = (_randn(g, t, c["experts"]) + 0.5 * _randn(g, c["experts"])).to(dt).requires_grad_(train)
        s["bias"] = 0.05 * _randn(g, c["experts"]) if c["bias"] else None
        if train:
            s["dweights"] = _randn(g, t, c["topk"])
        return s
    s["idx"], s["weights"] = _routing(c, g)
    s["x"] = _randn(g, t, h, dtype=dt)
    s["scales"] = torch.rand(t, h // 128, device=DEV, generator=g) + 0.5 if c["dtype"] == "e4m3" else None
    s["results"] = _randn(g, t * c["topk"], h, dtype=torch.bfloat16 if c["dtype"] == "e4m3" else dt)
    if train:
        s["drows"], s["dout"] = _randn(g, t * c["topk"], h, dtype=dt), _randn(g, t, h, dtype=dt)
        for name in ("x", "results", "weights"):
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------
def _sum(st):
    """The residual's addition, rounded to the residual's type; the rows themselves without one."""
    x, r = st["x"].detach(), st["residual"]
    return x if r is None else (x.float() + r.detach().float()).to(r.dtype)


def _plain_norm(st):
    c, w, dt = st["case"], st["weight"].detach().float(), st["x"].dtype
    total = _sum(st)
    s = total.float()
    rstd = torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)
    hat = s * rstd
    y = hat * w
    if c["op"] == "norm":
        return {"rows": y.to(dt), "sum": total}
    if c["op"] == "norm_quant":
        out = {} if st["residual"] is None else {"sum": total}
        if c["mode"] == 2:
            inv = 127.0 / (y.abs().amax(-1, keepdim=True) + 1e-12)
            code = torch.round(y * inv).clamp(-127, 127)
            return dict(out, values=(code / inv).to(torch.bfloat16), scales=(1.0 / inv).squeeze(-1))
        v = y.unflatten(-1, (-1, 128))
        amax = v.abs().amax(-1, keepdim=True).clamp(min=1e-4)
        scale = amax / 448.0
        if c["mode"] == 4:
            m, ex = torch.frexp(scale)
            scale = torch.ldexp(torch.ones_like(m), ex - (m == 0.5).int())
        q = (v / scale).clamp(-448, 448).flatten(-2).to(torch.float8_e4m3fn)
        return dict(out, codes=q, scales=scale.squeeze(-1).to(torch.float8_e8m0fnu if c["mode"] == 4 else torch.float32))
    dy, ds = st["dy"].float(), st["dsum"].float()
    p = dy * w
    d = ds + rstd * (p - hat * (p * hat).mean(-1, keepdim=True))
    return {"rows": y.to(dt), "sum": total, "dx": d.to(dt), "dresidual": d.to(total.dtype), "dweight": (dy * hat).sum(0).to(dt)}


def _plain_route(st):
    c, logits, bias = st["case"], st["logits"].detach(), st["bias"]
    t, e, k = c["tokens"], c["experts"], c["topk"]
    x = logits.double()  # choices lie next to borders
    if c["score"] == "softmax":
        p = torch.exp(x - x.amax(-1, keepdim=True))
        score = p / p.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    rank = x if bias is None else score + bias.double()
    if c["topk_groups"] < c["groups"]:
        best = torch.sort((score if bias is None else rank).view(t, c["groups"], -1), dim=-1, descending=True, stable=True).values
        best = best[..., : 2 if c["score"] == "sigmoid" else 1].sum(-1)
        keep = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, : c["topk_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True)
        rank = torch.where(open_.repeat_interleave(e // c["groups"], 1), rank, torch.full_like(rank, -math.inf))
    idx = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :k]
    s = torch.gather(score, 1, idx)
    total = s.sum(-1, keepdim=True)
    w = s / total if c["renorm"] else s
    w = w * _scale(c)
    if c["op"] == "route":
        return {"idx": idx, "weights": w.float()}
    g = st["dweights"].double() * _scale(c)
    ds = (g - (g * s / total).sum(-1, keepdim=True)) / total if c["renorm"] else g
    if c["score"] == "softmax":
        full = torch.zeros_like(score).scatter_(1, idx, ds)
        d = score * (full - (full * score).sum(-1, keepdim=True))
    else:
        d = torch.zeros_like(score).scatter_(1, idx, ds * s * (1 - s))
    return {"idx": idx, "weights": w.float(), "dlogits": d.to(logits.dtype)}


def _scale(c):
    return 2.5 if c["score"] == "sigmoid" else 1.0


def _plain_regroup(st):
    c, idx, x = st["case"], st["idx"], st["x"].detach()
    t, k, e, h = c["tokens"], c["topk"], c["experts"], c["hidden"]
    flat = idx.reshape(-1)
    live = flat >= 0
    key = torch.where(live, flat, torch.full_like(flat, e))
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(e + 1, dtype=torch.long, device=DEV).scatter_add_(0, key, torch.ones_like(key))
    ends = torch.cat([torch.zeros_like(counts[:1]), counts[:e].cumsum(0)])
    place = torch.empty_like(flat)
    place[order] = torch.arange(t * k, device=DEV)
    slots = torch.where(live, place, torch.full_like(place, -1)).view(t, k)
    used = (torch.arange(t * k, device=DEV) < ends[-1])[:, None]
    rows = torch.where(used, x.float()[order // k], torch.zeros((), device=DEV)).to(x.dtype)
    z, w = st["results"].detach().float(), st["weights"].detach()
    pick = z[slots.clamp(min=0).reshape(-1)].view(t, k, h)
    w0 = torch.where(slots >= 0, w, torch.zeros_like(w))
    out = {"rows": rows, "offsets": ends.int(), "slots": slots.int(), "out": (pick * w0[..., None]).sum(1).to(st["results"].dtype)}
    if st["scales"] is not None:
        out["scales"] = torch.where(used, st["scales"][order // k], torch.zeros((), device=DEV))
    if c["op"] == "regroup":
        return out
    dr = st["drows"].float()[slots.clamp(min=0).reshape(-1)].view(t, k, h)
    dout = st["dout"].float()
    out["dx"] = torch.where((slots >= 0)[..., None], dr, torch.zeros((), device=DEV)).sum(1).to(x.dtype)
    dz = dout[order // k] * w0.reshape(-1)[order][:, None]
    out["dresults"] = torch.where(used, dz, torch.zeros((), device=DEV)).to(x.dtype)
    out["dweights"] = torch.where(slots >= 0, (pick * dout[:, None]).sum(-1), torch.zeros((), device=DEV))
    return out


# ------------------------------------------------------------------------------------------------
# The library's calls
# ------------------------------------------------------------------------------------------------
def _run_own(st):
    from umdk_original_b200 import ops

    c = st["case"]
    if c["op"] == "norm":
        y, total = ops.add_rms_norm(st["x"], st["residual"], st["weight"], EPS)
        return {"rows": y, "sum": total}
    if c["op"] == "norm_train":
        y, total = ops.add_rms_norm(st["x"], st["residual"], st["weight"], EPS)
        dx, dr, dw = torch.autograd.grad((y, total), (st["x"], st["residual"], st["weight"]), (st["dy"], st["dsum"]))
        return {"rows": y.detach(), "sum": total.detach(), "dx": dx, "dresidual": dr, "dweight": dw}
    if c["op"] == "norm_quant":
        q, s, total, _ = ops.rms_norm_quant(st["x"], st["weight"], c["mode"], st["residual"], EPS)
        out = {} if st["residual"] is None else {"sum": total}
        if c["mode"] == 2:
            return dict(out, values=torch.mul(q, s[:, None], out=torch.empty_like(q, dtype=torch.bfloat16)), scales=s)
        return dict(out, codes=q, scales=s.to(torch.float8_e8m0fnu) if c["mode"] == 4 else s)
    if c["op"].startswith("route"):
        idx, w = ops.moe_route(st["logits"], c["topk"], st["bias"], c["score"], c["groups"], c["topk_groups"],
                               2 if c["score"] == "sigmoid" else 1, c["renorm"], _scale(c))
        if c["op"] == "route":
            return {"idx": idx, "weights": w}
        (d,) = torch.autograd.grad(w, st["logits"], st["dweights"])
        return {"idx": idx, "weights": w.detach(), "dlogits": d}
    rows, scales, offsets, slots = ops.moe_group_rows(st["x"], st["idx"], c["experts"], st["scales"])
    out = ops.moe_ungroup_rows(st["results"], slots, st["weights"])
    got = {"rows": rows.detach(), "offsets": offsets, "slots": slots, "out": out.detach()}
    if st["scales"] is not None:
        got["scales"] = scales
    if c["op"] == "regroup_train":
        got["dx"], got["dresults"], got["dweights"] = torch.autograd.grad(
            (rows, out), (st["x"], st["results"], st["weights"]), (st["drows"], st["dout"]))
    return got


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    return _plain_norm(st) if op.startswith("norm") else _plain_route(st) if op.startswith("route") else _plain_regroup(st)


# ------------------------------------------------------------------------------------------------
# Results in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_norm(c, st):
    x, w = st["x"].detach().double(), st["weight"].detach().double()
    total = x if st["residual"] is None else (x + st["residual"].detach().double()).to(st["residual"].dtype).double()
    length = torch.sqrt(torch.linalg.vecdot(total, total) / c["hidden"] + EPS)[:, None]
    unit = total / length
    if c["op"] == "norm":
        return {"rows": unit * w, "sum": total}
    if c["op"] == "norm_train":
        dy, ds = st["dy"].double(), st["dsum"].double()
        along = torch.linalg.vecdot(dy * w, unit)[:, None] / c["hidden"]
        d = ds + (dy * w - along * unit) / length
        return {"rows": unit * w, "sum": total, "dx": d, "dresidual": d, "dweight": torch.einsum("th,th->h", dy, unit)}
    y = unit * w
    out = {} if st["residual"] is None else {"sum": total}
    if c["mode"] == 2:
        return dict(out, values=y, scales=(y.abs().max(-1).values + 1e-12) / 127)
    top = y.view(c["tokens"], -1, 128).abs().max(-1).values.clamp(min=1e-4) / 448
    if c["mode"] == 4:
        top = torch.exp2(torch.ceil(torch.log2(top)))
    return dict(out, codes=y / top.repeat_interleave(128, -1), scales=top)


def _exact_route(c, st):
    x = st["logits"].detach().double()
    t, e, k = c["tokens"], c["experts"], c["topk"]
    s = torch.softmax(x, -1) if c["score"] == "softmax" else torch.sigmoid(x)
    by = x if st["bias"] is None else s + st["bias"].double()
    if c["topk_groups"] < c["groups"]:
        of_group = (s if st["bias"] is None else by).reshape(t, c["groups"], -1)
        two = torch.topk(of_group, 2 if c["score"] == "sigmoid" else 1, -1).values.sum(-1)
        # a group is out if as many as may stay are before it
        before = (two[:, None, :] > two[:, :, None]).sum(-1) + ((two[:, None, :] == two[:, :, None]) & torch.ones(c["groups"], c["groups"], device=DEV).tril(-1).bool()).sum(-1)
        by = by.reshape(t, c["groups"], -1).masked_fill((before >= c["topk_groups"])[..., None], -math.inf).reshape(t, e)
    left, picks = by.clone(), []
    for _ in range(k):
        top = left.max(-1, keepdim=True).values
        pick = (left == top).int().argmax(-1, keepdim=True)  # the first of equals
        picks.append(pick)
        left.scatter_(1, pick, -math.inf)
    idx = torch.cat(picks, 1)
    chosen = s.gather(1, idx)
    scale = 2.5 if c["score"] == "sigmoid" else 1.0
    w = scale * (chosen / chosen.sum(-1, keepdim=True) if c["renorm"] else chosen)
    if c["op"] == "route":
        return {"idx": idx, "weights": w}
    g, share, d = st["dweights"].double(), w, torch.zeros_like(x)
    if c["renorm"]:  # of w = scale s / sum s, by the logarithmic derivatives of s
        log_grad = share * (g - (g * share).sum(-1, keepdim=True) / scale)
    else:
        log_grad = g * share
    if c["score"] == "sigmoid":
        d.scatter_(1, idx, log_grad * torch.sigmoid(-x.gather(1, idx)))
    else:
        d = d.scatter_(1, idx, log_grad) - s * log_grad.sum(-1, keepdim=True)
    return {"idx": idx, "weights": w, "dlogits": d}


def _exact_regroup(c, st):
    t, k, e = c["tokens"], c["topk"], c["experts"]
    idx = st["idx"].cpu()
    lists = [torch.nonzero(idx.reshape(-1) == j).flatten() for j in range(e)]
    pairs = torch.cat(lists)
    offsets = torch.tensor([0] + [len(v) for v in lists]).cumsum(0).int()
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    slots[pairs] = torch.arange(len(pairs), dtype=torch.int32)
    pairs = pairs.to(DEV)
    n = len(pairs)
    rows = torch.zeros(t * k, c["hidden"], device=DEV, dtype=torch.float64)
    rows[:n] = st["x"].detach().double()[pairs // k]
    z, w = st["results"].detach().double(), st["weights"].detach().double().reshape(-1)[pairs]
    out = torch.zeros(t, c["hidden"], device=DEV, dtype=torch.float64).index_add_(0, pairs // k, z[:n] * w[:, None])
    got = {"rows": rows, "offsets": offsets, "slots": slots.view(t, k), "out": out}
    if st["scales"] is not None:
        got["scales"] = torch.zeros(t * k, st["scales"].shape[1], device=DEV, dtype=torch.float64)
        got["scales"][:n] = st["scales"].double()[pairs // k]
    if c["op"] == "regroup_train":
        got["dx"] = torch.zeros_like(out).index_add_(0, pairs // k, st["drows"].double()[:n])
        dout = st["dout"].double()[pairs // k]
        got["dresults"] = torch.zeros_like(rows)
        got["dresults"][:n] = dout * w[:, None]
        got["dweights"] = torch.zeros(t * k, device=DEV, dtype=torch.float64)
        got["dweights"][pairs] = torch.linalg.vecdot(dout, z[:n])
        got["dweights"] = got["dweights"].view(t, k)
    return got


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    return _exact_norm(case, st) if op.startswith("norm") else _exact_route(case, st) if op.startswith("route") else _exact_regroup(case, st)
