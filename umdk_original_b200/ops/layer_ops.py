"""Operators round the experts that need no ``Buffer``: schemas and CPU implementations.

``rms_norm`` / ``add_rms_norm``: root-mean-square norm of rows, of ``x`` or of ``x + residual``; differentiable.  The sum is rounded to
the residual's type, and it is the rounded sum that is normalised.  ``rms_norm_quant``: the same with rows in 8 bits, in the quant modes
of the dispatch.  ``moe_route``: experts and weights of every token from its logits; differentiable in the logits.
``moe_group_rows`` / ``moe_ungroup_rows``: rows of tokens sorted by expert, in the form that ``grouped_mlp`` and the grouped products
take, and the experts' results brought back; differentiable.  What dispatch and combine do for a group of ranks, these do for one
rank, without a ``Buffer``.

The CUDA implementations live in csrc/bindings_layer.cpp; the CPU ones here follow the same contracts.
"""
from __future__ import annotations

from typing import Tuple

import torch

from . import reference as ref

SCHEMAS = [
    "rms_norm(Tensor x, Tensor weight, float eps=1e-6) -> Tensor",
    "add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps=1e-6) -> (Tensor, Tensor)",
    "rms_norm_train(Tensor x, Tensor? residual, Tensor weight, float eps=1e-6) -> (Tensor, Tensor, Tensor)",
    "rms_norm_backward(Tensor dy, Tensor? dsum, Tensor sum, Tensor weight, Tensor rstd, bool need_dx=True, bool need_dresidual=True, "
    "bool need_dweight=True) -> (Tensor, Tensor, Tensor)",
    "rms_norm_quant(Tensor x, Tensor weight, int quant_mode, Tensor? residual=None, float eps=1e-6, bool with_rows=False) -> "
    "(Tensor, Tensor, Tensor, Tensor)",
    "moe_route(Tensor logits, int k, Tensor? bias=None, str score=\"softmax\", int num_groups=1, int topk_groups=1, int group_top=1, "
    "bool renormalize=True, float scale=1.0) -> (Tensor, Tensor)",
    "moe_route_backward(Tensor dweights, Tensor logits, Tensor topk_idx, str score=\"softmax\", bool renormalize=True, float scale=1.0) "
    "-> Tensor",
    "moe_group_rows(Tensor x, Tensor topk_idx, int num_experts, Tensor? scales=None) -> (Tensor, Tensor, Tensor, Tensor)",
    "moe_ungroup_rows(Tensor rows, Tensor slots, Tensor? topk_weights=None, Tensor? residual=None) -> Tensor",
    "moe_ungroup_rows_backward(Tensor dout, Tensor rows, Tensor slots, Tensor? topk_weights=None, bool need_drows=True, "
    "bool need_dweights=True) -> (Tensor, Tensor)",
]

MAX_HIDDEN, MAX_EXPERTS, MAX_TOPK, MAX_GROUPS = 16384, 1024, 32, 32
FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_PREFIX = "umdk_cam_op_lib: "


def _check(cond: bool, message: str) -> None:
    if not cond:
        raise RuntimeError(_PREFIX + message)


def _check_float(t: torch.Tensor, what: str) -> None:
    _check(t.dtype in FLOATS, f"{what} must be bfloat16, float16 or float32")


def _contiguous(*tensors) -> None:
    for t, what in tensors:
        _check(t is None or t.is_contiguous(), f"{what} must be contiguous")


# ------------------------------------------------------------------------------------------------
# Norm
# ------------------------------------------------------------------------------------------------
def _check_norm(op: str, x, residual, weight, eps: float) -> None:
    _contiguous((x, "x"), (weight, "weight"), (residual, "residual"))
    _check_float(x, "x")
    _check(x.dim() >= 1 and x.shape[-1] >= 1, f"{op}: x must be [..., h]")
    h = x.shape[-1]
    _check(h <= MAX_HIDDEN, f"{op}: rows of {h} values; at most {MAX_HIDDEN}")
    _check(weight.dim() == 1 and weight.shape[0] == h and weight.dtype in (x.dtype, torch.float32),
           f"{op}: weight must be [{h}] of x's type or float32")
    _check(eps >= 0, f"{op}: eps must not be negative")
    _check(residual is None or (residual.shape == x.shape and residual.dtype in (x.dtype, torch.float32)),
           f"{op}: residual must be {list(x.shape)} of x's type or float32")


def _norm(x, residual, weight, eps: float):
    """(y in fp32, the stored sum or x, rstd)"""
    total = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    s = total.float()
    rstd = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    return s * rstd * weight.float(), total, rstd


def rms_norm_train_cpu(x, residual, weight, eps=1e-6):
    _check_norm("rms_norm_train", x, residual, weight, eps)
    y, total, rstd = _norm(x, residual, weight, eps)
    return y.to(x.dtype), x.new_empty(0) if residual is None else total, rstd.reshape(-1)


def rms_norm_cpu(x, weight, eps=1e-6):
    _check_norm("rms_norm", x, None, weight, eps)
    return _norm(x, None, weight, eps)[0].to(x.dtype)


def add_rms_norm_cpu(x, residual, weight, eps=1e-6):
    _check_norm("add_rms_norm", x, residual, weight, eps)
    y, total, _ = _norm(x, residual, weight, eps)
    return y.to(x.dtype), total


def rms_norm_backward_cpu(dy, dsum, sum, weight, rstd, need_dx=True, need_dresidual=True, need_dweight=True):
    _check_norm("rms_norm_backward", dy, sum, weight, 0.0)
    _contiguous((rstd, "rstd"), (dsum, "dsum"))
    _check(rstd.dtype == torch.float32 and rstd.numel() == dy.numel() // dy.shape[-1],
           "rms_norm_backward: rstd must be float32 with one value per row")
    _check(dsum is None or (dsum.shape == sum.shape and dsum.dtype == sum.dtype), "rms_norm_backward: dsum must be like sum")
    hat = sum.float() * rstd.view(*dy.shape[:-1], 1)
    p = dy.float() * weight.float()
    d = rstd.view(*dy.shape[:-1], 1) * (p - hat * (p * hat).mean(-1, keepdim=True))
    if dsum is not None:
        d = d + dsum.float()
    one = dy.dtype == sum.dtype
    dw = (dy.float() * hat).reshape(-1, dy.shape[-1]).sum(0).to(weight.dtype) if need_dweight else weight.new_empty(0)
    return (d.to(dy.dtype) if need_dx or (one and need_dresidual) else dy.new_empty(0),
            d.to(sum.dtype) if need_dresidual and not one else sum.new_empty(0), dw)


def rms_norm_quant_cpu(x, weight, quant_mode, residual=None, eps=1e-6, with_rows=False):
    _check_norm("rms_norm_quant", x, residual, weight, eps)
    _check(quant_mode in (2, 3, 4), f"rms_norm_quant: quant_mode must be 2 (int8), 3 (e4m3) or 4 (e4m3, power-of-two scales), got {quant_mode}")
    h = x.shape[-1]
    _check(quant_mode == 2 or h % 128 == 0, f"rms_norm_quant: e4m3 rows must be a multiple of 128 values, not {h}")
    y, total, _ = _norm(x, residual, weight, eps)
    flat = y.reshape(-1, h)
    if quant_mode == 2:
        q, s = ref.quant_int8_token(flat)
        s = s.view(x.shape[:-1])
    else:
        q, s = ref.quant_fp8_1x128(flat, quant_mode == 4)
        s = torch.where(flat.view(-1, h // 128, 128).isnan().any(-1), torch.full_like(s, float("nan")), s)  # rounding up to a power of two loses it
        s = s.view(*x.shape[:-1], h // 128)
    return q.view(x.shape), s, x.new_empty(0) if residual is None else total, y.to(x.dtype) if with_rows else x.new_empty(0)


# ------------------------------------------------------------------------------------------------
# Routing
# ------------------------------------------------------------------------------------------------
def _check_logits(op: str, logits, k: int) -> None:
    _contiguous((logits, "logits"))
    _check_float(logits, "logits")
    _check(logits.dim() == 2, f"{op}: logits must be [T, E]")
    _check(1 <= k <= min(logits.shape[1], MAX_TOPK), f"{op}: k {k} outside [1, min({logits.shape[1]} experts, {MAX_TOPK})]")
    _check(logits.shape[1] <= MAX_EXPERTS, f"{op}: logits {list(logits.shape)}; at most {MAX_EXPERTS} experts")


def _check_score(score: str) -> None:
    _check(score in ("softmax", "sigmoid"), f"moe_route: score must be 'softmax' or 'sigmoid', got '{score}'")


def _scores(x: torch.Tensor, score: str) -> torch.Tensor:
    return torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1)


def moe_route_cpu(logits, k, bias=None, score="softmax", num_groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
    _check_logits("moe_route", logits, k)
    _check_score(score)
    _contiguous((bias, "bias"))
    t, e = logits.shape
    _check(bias is None or (bias.dtype == torch.float32 and tuple(bias.shape) == (e,)), f"moe_route: bias must be float32 [{e}]")
    _check(1 <= num_groups <= MAX_GROUPS and e % num_groups == 0,
           f"moe_route: {e} experts in {num_groups} groups; at most {MAX_GROUPS} groups of equal size")
    _check(1 <= topk_groups <= num_groups, f"moe_route: topk_groups {topk_groups} outside [1, {num_groups}]")
    _check(k <= e // num_groups * topk_groups, f"moe_route: k {k} of the {e // num_groups * topk_groups} experts in {topk_groups} groups")
    _check(group_top in (1, 2), f"moe_route: group_top must be 1 or 2, got {group_top}")
    x = logits.double()
    low = torch.full_like(x, float("-inf"))
    s = _scores(x, score)
    rank = x if bias is None else s + bias.double()
    closed = ~(x > float("-inf")) | ~(rank > float("-inf"))  # NaN too
    rank = torch.where(closed, low, rank)
    if topk_groups < num_groups:
        value = torch.where(closed, low, s if bias is None and group_top == 2 else rank).nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
        best = value.view(t, num_groups, -1).sort(-1, descending=True).values[..., :group_top]
        best = torch.where(best[..., :1] > float("-inf"), best.masked_fill(best == float("-inf"), 0.0).sum(-1, keepdim=True), best[..., :1]).squeeze(-1)
        top = best.sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        open_ = torch.zeros(t, num_groups, dtype=torch.bool).scatter_(1, top, True) & (best > float("-inf"))
        rank = torch.where(open_.repeat_interleave(e // num_groups, 1), rank, low)
    value, idx = rank.sort(dim=-1, descending=True, stable=True)
    empty = value[:, :k] == float("-inf")
    idx = idx[:, :k].masked_fill(empty, -1).contiguous()
    l = torch.where(empty, low[:, :k], x.gather(1, idx.clamp(min=0)))
    if renormalize:
        # relative to the largest chosen one: scores that underflow keep their ratios
        m = l.amax(-1, keepdim=True)
        w = torch.exp(l.clamp(max=0) - m.clamp(max=0)) / (1 + torch.exp(-l.abs())) if score == "sigmoid" else torch.exp(l - m)
        w = torch.where(empty, torch.zeros_like(w), w)
        w = torch.where(empty, torch.zeros_like(w), w / w.sum(-1, keepdim=True))
    else:
        w = torch.where(empty, torch.zeros_like(l), s.gather(1, idx.clamp(min=0)))
    bad = logits.isnan() if score == "sigmoid" else logits.isnan() | (x == float("inf"))
    w = torch.where(bad.any(-1, keepdim=True), torch.full_like(w, float("nan")), w * scale)
    return idx, w.float()


def moe_route_backward_cpu(dweights, logits, topk_idx, score="softmax", renormalize=True, scale=1.0):
    _check(topk_idx.dim() == 2, "moe_route_backward: topk_idx must be int64 [T, k]")
    _check_logits("moe_route_backward", logits, topk_idx.shape[1])
    _contiguous((dweights, "dweights"), (topk_idx, "topk_idx"))
    _check(topk_idx.dtype == torch.int64 and topk_idx.shape[0] == logits.shape[0], "moe_route_backward: topk_idx must be int64 [T, k]")
    _check(dweights.dtype == torch.float32 and dweights.shape == topk_idx.shape, "moe_route_backward: dweights must be float32 [T, k]")
    _check_score(score)
    x = logits.double()
    valid = (topk_idx >= 0) & (topk_idx < logits.shape[1])
    idx = topk_idx.clamp(0, logits.shape[1] - 1)
    g = torch.where(valid, dweights.double() * scale, torch.zeros(()).double())
    l = torch.where(valid, x.gather(1, idx), torch.full((), float("-inf")).double())
    d = torch.zeros_like(x)
    if renormalize:
        m = l.amax(-1, keepdim=True)
        q = torch.exp(l.clamp(max=0) - m.clamp(max=0)) / (1 + torch.exp(-l.abs())) if score == "sigmoid" else torch.exp(l - m)
        q = torch.where(valid, q, torch.zeros_like(q))
        q = torch.where(valid, q / q.sum(-1, keepdim=True), q)
        on = (g - (g * q).sum(-1, keepdim=True)) * q
        if score == "sigmoid":
            on = on * torch.sigmoid(-l)
    else:
        s = _scores(x, score)
        q = torch.where(valid, s.gather(1, idx), torch.zeros_like(l))
        on = g * q * (torch.sigmoid(-l) if score == "sigmoid" else 1)
        if score == "softmax":
            d = torch.where(x.amax(-1, keepdim=True) > float("-inf"), -s * (g * q).sum(-1, keepdim=True), d)
    d.scatter_add_(1, idx, torch.where(valid, on, torch.zeros_like(on)))
    return d.to(logits.dtype)


# ------------------------------------------------------------------------------------------------
# Rows grouped by expert and brought back
# ------------------------------------------------------------------------------------------------
def moe_group_rows_cpu(x, topk_idx, num_experts, scales=None):
    _contiguous((x, "x"), (topk_idx, "topk_idx"), (scales, "scales"))
    _check(x.dim() == 2 and x.shape[1] >= 1 and topk_idx.dim() == 2 and topk_idx.shape[0] == x.shape[0], "moe_group_rows: x must be [T, h], topk_idx [T, k]")
    _check(x.dtype in (*FLOATS, torch.float8_e4m3fn, torch.int8),
           "moe_group_rows: x (where it is not float8_e4m3fn or int8) must be bfloat16, float16 or float32")
    _check(topk_idx.dtype in (torch.int64, torch.int32), "moe_group_rows: topk_idx must be int64 or int32")
    t, k = topk_idx.shape
    _check(1 <= k <= MAX_TOPK, f"moe_group_rows: {k} choices per token; 1 to {MAX_TOPK}")
    _check(1 <= num_experts <= MAX_EXPERTS, f"moe_group_rows: {num_experts} experts; 1 to {MAX_EXPERTS}")
    _check(scales is None or (scales.dtype == torch.float32 and scales.dim() in (1, 2) and scales.shape[0] == t and (scales.dim() == 1 or scales.shape[1] >= 1)), "moe_group_rows: scales must be float32 [T] or [T, s]")
    ids = topk_idx.reshape(-1).long()
    ids = torch.where((ids >= 0) & (ids < num_experts), ids, torch.full_like(ids, num_experts))
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=num_experts + 1)[:num_experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    n = int(offsets[-1])
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    slots[order[:n]] = torch.arange(n, dtype=torch.int32)
    token = order[:n] // k

    def moved(v):
        if t == 0:
            return v.new_empty(v.shape)
        bytes_ = v.view(torch.uint8).view(t, -1)  # indexing does not know every type
        out = torch.zeros(t * k, bytes_.shape[1], dtype=torch.uint8)
        out[:n] = bytes_[token]
        return out.view(v.dtype).view(t * k, *v.shape[1:])
    rows, row_scales = moved(x), torch.empty(0) if scales is None else moved(scales)
    return rows, row_scales, offsets.to(torch.int32), slots.view(t, k)


def _check_ungroup(op: str, rows, slots, weights, numbered: bool = False) -> None:
    _contiguous((rows, "rows"), (slots, "slots"), (weights, "topk_weights"))
    _check_float(rows, "rows")
    _check(rows.dim() == 2 and (rows.shape[1] >= 1 or numbered), f"{op}: rows must be [M, h]")
    _check(slots.dim() == 2 and slots.dtype == torch.int32 and 1 <= slots.shape[1] <= MAX_TOPK, f"{op}: slots must be int32 [T, k] with k of 1 to {MAX_TOPK}")
    _check(weights is None or (weights.dtype == torch.float32 and weights.shape == slots.shape), f"{op}: topk_weights must be float32 {list(slots.shape)}")


def _picked(rows, slots, weights) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(slots in range, the rows they name in fp32 [T, k, h], weights with zeros elsewhere)"""
    valid = (slots >= 0) & (slots < rows.shape[0])
    at = torch.where(valid, slots, torch.zeros_like(slots)).long()
    picked = rows.float()[at] if rows.shape[0] else torch.zeros(*slots.shape, rows.shape[1])
    w = torch.ones(slots.shape) if weights is None else weights
    return valid, torch.where(valid[..., None], picked, torch.zeros(())), torch.where(valid, w, torch.zeros(()))


def moe_ungroup_rows_cpu(rows, slots, topk_weights=None, residual=None):
    _check_ungroup("moe_ungroup_rows", rows, slots, topk_weights)
    _contiguous((residual, "residual"))
    _check(residual is None or (residual.dtype == rows.dtype and tuple(residual.shape) == (slots.shape[0], rows.shape[1])),
           "moe_ungroup_rows: residual must be [T, h] of the rows' type")
    _, picked, w = _picked(rows, slots, topk_weights)
    out = (picked * w[..., None]).sum(1)
    return (out if residual is None else out + residual.float()).to(rows.dtype)


def moe_ungroup_rows_backward_cpu(dout, rows, slots, topk_weights=None, need_drows=True, need_dweights=True):
    op = "moe_ungroup_rows_backward"
    # gradients of rows alone need their number: rows [M, 0] will do
    numbered = not need_dweights and rows.dim() == 2 and rows.shape[1] == 0 and dout.dim() == 2 and dout.shape[1] >= 1
    _check_ungroup(op, rows, slots, topk_weights, numbered)
    _contiguous((dout, "dout"))
    h = dout.shape[1] if numbered else rows.shape[1]
    _check(dout.dtype == rows.dtype and tuple(dout.shape) == (slots.shape[0], h), f"{op}: dout must be [T, h] of the rows' type")
    valid, picked, w = _picked(rows, slots, topk_weights)
    d = dout.float()
    drows, dw = rows.new_empty(0), torch.empty(0)
    if need_drows:
        named = slots[valid]
        _check(named.unique().numel() == named.numel(), f"{op}: a row belongs to one slot at most")
        drows = torch.zeros(rows.shape[0], h, dtype=torch.float32)
        drows[slots[valid].long()] = (d[:, None] * w[..., None])[valid]
        drows = drows.to(rows.dtype)
    if need_dweights:
        dw = torch.where(valid, (picked * d[:, None]).sum(-1), torch.zeros(()))
    return drows, dw


CPU_IMPLS = {
    "rms_norm": rms_norm_cpu,
    "add_rms_norm": add_rms_norm_cpu,
    "rms_norm_train": rms_norm_train_cpu,
    "rms_norm_backward": rms_norm_backward_cpu,
    "rms_norm_quant": rms_norm_quant_cpu,
    "moe_route": moe_route_cpu,
    "moe_route_backward": moe_route_backward_cpu,
    "moe_group_rows": moe_group_rows_cpu,
    "moe_ungroup_rows": moe_ungroup_rows_cpu,
    "moe_ungroup_rows_backward": moe_ungroup_rows_backward_cpu,
}
