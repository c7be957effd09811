"""Definitions in 64 bits and error bounds for the tests of norm, routing and rows grouped by expert (CPU and GPU).

u = 2^-24 is half a step of fp32, relative; a result of 16 bits is rounded once more, by half a step of its type."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    """(relative, absolute) error of one rounding: fp16 has subnormals within reach, whose half step is 2^-25."""
    return (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2), (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130)


def within(got, want, tol, what=""):
    """Every value inside its bound; NaN and infinities at the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~want.isfinite()
    assert torch.equal(got[odd].nan_to_num(7.0, 8.0, 9.0), want[odd].nan_to_num(7.0, 8.0, 9.0)), what
    bad = ~((got - want).abs() <= tol) & ~odd
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / tol.clamp(min=1e-300))[bad].max()))


def norm64(x, residual, weight, eps):
    """(y, the stored sum, 1 / rms)"""
    total = x if residual is None else (x.double() + residual.double()).to(residual.dtype)
    s = total.double()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s * rstd * weight.double(), total, rstd


def norm_tol(y, dtype):
    # sum of squares: 32 additions in a thread, 10 between threads, the squares: 43 u, half of it in 1 / rms, with the division, the
    # root and the addition of eps 26 u; two products: below 32 u
    half, tiny = half_step(dtype)
    return y.abs() * (half + 32 * U) + tiny


def norm_grads64(dy, dsum, total, weight, eps):
    s, w, g = total.double(), weight.double(), dy.double()
    h = s.shape[-1]
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    hat, p = s * rstd, g * w
    along = (p * hat).sum(-1, keepdim=True) / h
    ds = torch.zeros_like(s) if dsum is None else dsum.double()
    d = ds + rstd * (p - hat * along)
    size = ds.abs() + rstd * (p.abs() + hat.abs() * (p * hat).abs().sum(-1, keepdim=True) / h)
    flat = (g * hat).reshape(-1, h)
    return d, size, flat.sum(0), flat.abs().sum(0)


def norm_grad_tol(d, size, dtype):
    # 1 / rms 28 u; a product of the sum 31 u, its additions 26 u, so the sum 58 u; times hat 29 u more; the rest 30 u: below 128 u
    half, tiny = half_step(dtype)
    return d.abs() * half + size * (128 * U) + tiny


def weight_grad_tol(dw, size, rows, dtype):
    # a product 30 u; at most as many additions as rows and 64 to join blocks and warps
    half, tiny = half_step(dtype)
    return dw.abs() * half + size * ((rows + 96) * U) + tiny


def route64(logits, k, bias=None, score="softmax", num_groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
    """One row at a time, in plain Python order: lowest index first among equals."""
    x = logits.double().cpu()
    t, e = x.shape
    s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
    rank = x if bias is None else s + bias.double().cpu()
    idx = torch.full((t, k), -1, dtype=torch.int64)
    w = torch.zeros(t, k, dtype=torch.float64)
    inf = float("inf")
    for r in range(t):
        ok = [j for j in range(e) if x[r, j] > -inf and rank[r, j] > -inf]
        if topk_groups < num_groups:
            n = e // num_groups
            value = rank[r] if bias is not None or group_top == 1 else s[r]
            worth = {}
            for g in range(num_groups):
                best = sorted((float(value[j]) for j in ok if j // n == g), reverse=True)[:group_top]
                if best:
                    worth[g] = sum(best)
            open_ = sorted(worth, key=lambda g: (-worth[g], g))[:topk_groups]
            ok = [j for j in ok if j // n in open_]
        chosen = sorted(ok, key=lambda j: (-float(rank[r, j]), j))[:k]
        for j, c in enumerate(chosen):
            idx[r, j] = c
            if renormalize:
                # s_c / sum s = 1 / sum of the ratios, by the logarithms of the scores
                log = torch.log_softmax(x[r], -1) if score == "softmax" else torch.nn.functional.logsigmoid(x[r])
                w[r, j] = scale / torch.exp(log[chosen] - log[c]).sum()
            else:
                w[r, j] = scale * s[r, c]
        if x[r].isnan().any():
            w[r] = float("nan")
    return idx.to(logits.device), w.to(logits.device)


def route_weight_tol(w):
    # expf 2 u with an argument of up to 30 that is itself rounded (30 u), a sum of 32 terms in a lane and 5 between lanes, two divisions,
    # the scale: below 128 u
    return w.abs() * (128 * U) + 2.0 ** -140


def route_grad64(dweights, logits, idx, score="softmax", renormalize=True, scale=1.0):
    """(gradient, size of its terms)"""
    x = logits.double()
    valid = idx >= 0
    at = idx.clamp(min=0)
    s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
    g = torch.where(valid, dweights.double() * scale, 0.0)
    q = torch.where(valid, s.gather(1, at), 0.0)
    if renormalize:
        q = q / q.sum(-1, keepdim=True).clamp(min=1e-300)
    other = torch.sigmoid(-x).gather(1, at) if score == "sigmoid" else torch.ones_like(q)
    d, size = torch.zeros_like(x), torch.zeros_like(x)
    if renormalize or score == "softmax":
        along, long = (g * q).sum(-1, keepdim=True), (g * q).abs().sum(-1, keepdim=True)
    else:
        along = long = torch.zeros_like(g[:, :1])
    if renormalize or score == "sigmoid":
        d.scatter_add_(1, at, torch.where(valid, (g - along) * q * other, 0.0))
        size.scatter_add_(1, at, torch.where(valid, (g.abs() + long) * q * other, 0.0))
    else:
        d = -s * along
        size = s * long
        d.scatter_add_(1, at, g * q)
        size.scatter_add_(1, at, (g * q).abs())
    return d, size


def group64(x, topk_idx, num_experts, scales=None):
    """rows, scales, offsets, slots by a loop over experts and pairs"""
    t, k = topk_idx.shape
    ids = topk_idx.reshape(-1).tolist()
    order = [p for e in range(num_experts) for p in range(t * k) if ids[p] == e]
    count = [sum(1 for i in ids if i == e) for e in range(num_experts)]
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    for r, p in enumerate(order):
        slots[p] = r
    rows = torch.zeros(t * k, *x.shape[1:], dtype=torch.float32, device=x.device)
    token = torch.tensor(order, dtype=torch.long, device=x.device) // k
    rows[: len(order)] = x.float()[token]
    rs = None
    if scales is not None:
        rs = torch.zeros(t * k, *scales.shape[1:], device=x.device)
        rs[: len(order)] = scales[token]
    off = torch.tensor([0] + count).cumsum(0).to(torch.int32)
    return rows, rs, off.to(x.device), slots.view(t, k).to(x.device)
