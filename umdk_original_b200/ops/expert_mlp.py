"""Expert-MLP operators that need no ``Buffer``: schemas and CPU implementations.

``quantize_fp4`` / ``dequantize_fp4`` / ``grouped_gemm_fp4`` / ``grouped_gemm_fp4_swiglu``: 4-bit floating point with block
scales (the formats are described in csrc/common/fp4.cuh).  The CUDA implementations live in csrc/bindings_expert.cpp; the CPU
ones here follow the same contracts in fp32, expert by expert.

``grouped_mlp``: the gated feed-forward block of 16-bit experts, differentiable in the rows and both weights.  Its parts,
``grouped_mlp_train`` (also returns what the backward pass needs: act, and the gate and up values in fp32) and
``grouped_mlp_backward``, can be called by programs that keep their own graph of derivatives.  Rows of no expert hold nothing
defined in act and in the gate and up values; the backward pass reads none of them.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

SCHEMAS = [
    "quantize_fp4(Tensor x, int block=16, Tensor? global_scale=None) -> (Tensor, Tensor)",
    "dequantize_fp4(Tensor q, Tensor s, Tensor? global_scale=None, ScalarType? dtype=None) -> Tensor",
    "grouped_gemm_fp4(Tensor a_q, Tensor a_s, Tensor w_q, Tensor w_s, Tensor expert_offsets, "
    "Tensor? a_global_scale=None, Tensor? w_global_scale=None) -> Tensor",
    "grouped_gemm_fp4_swiglu(Tensor a_q, Tensor a_s, Tensor w_q, Tensor w_s, Tensor expert_offsets, "
    "Tensor? a_global_scale=None, Tensor? w_global_scale=None, Tensor? out_global_scale=None) -> (Tensor, Tensor)",
    "grouped_mlp(Tensor x, Tensor w1, Tensor w2, Tensor expert_offsets) -> Tensor",
    "grouped_mlp_train(Tensor x, Tensor w1, Tensor w2, Tensor expert_offsets) -> (Tensor, Tensor, Tensor)",
    "grouped_mlp_backward(Tensor dy, Tensor x, Tensor w1, Tensor w2, Tensor expert_offsets, Tensor act, Tensor gate_up, "
    "bool need_dx=True, bool need_dw1=True, bool need_dw2=True) -> (Tensor, Tensor, Tensor)",
]

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_PREFIX = "umdk_cam_op_lib: "


def _check(cond: bool, message: str) -> None:
    if not cond:
        raise RuntimeError(_PREFIX + message)


def _block_of(s: torch.Tensor, what: str) -> int:
    _check(s.dtype in (torch.float8_e4m3fn, torch.float8_e8m0fnu),
           f"{what} must be float8_e4m3fn (nvfp4) or float8_e8m0fnu (mxfp4)")
    return 16 if s.dtype == torch.float8_e4m3fn else 32


def _check_gscale(g: Optional[torch.Tensor], block: int, per: int, what: str) -> None:
    if g is not None:
        _check(block == 16, f"{what}: mxfp4 has no global scale")
        _check(g.dtype == torch.float32 and g.numel() == max(per, 1), f"{what} must be float32 with {max(per, 1)} element(s)")


def _gscales_of(g: Optional[torch.Tensor], t: torch.Tensor) -> int:
    return t.shape[0] if g is not None and t.dim() == 3 and g.numel() != 1 else 0


def _check_fp4(q: torch.Tensor, s: torch.Tensor, block: int, what: str) -> int:
    _check(q.dtype == torch.uint8 and q.dim() >= 1, f"{what} codes must be uint8 [..., K / 2]")
    k = q.shape[-1] * 2
    _check(k % block == 0, f"{what}: K {k} is not a multiple of the block {block}")
    _check(tuple(s.shape) == (*q.shape[:-1], k // block), f"{what} scales must be [..., K / {block}] for codes [..., K / 2]")
    return k


def quantize_fp4_cpu(x: torch.Tensor, block: int = 16, global_scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    _check(block in (16, 32), f"block must be 16 (nvfp4) or 32 (mxfp4), got {block}")
    _check(x.is_contiguous(), "x must be contiguous")
    _check(x.dtype in (torch.bfloat16, torch.float16, torch.float32), "x must be bfloat16, float16 or float32")
    _check(x.dim() >= 1 and x.shape[-1] % block == 0 and x.shape[-1] > 0, f"quantize_fp4: the last dimension must be a multiple of {block}")
    per = _gscales_of(global_scale, x)
    _check_gscale(global_scale, block, per, "global_scale")
    v = x.float().unflatten(-1, (-1, block))
    amax = v.abs().amax(-1)
    if block == 16:
        g = torch.ones(1) if global_scale is None else global_scale.reshape(-1, *([1] * (amax.dim() - 1))) if per else global_scale
        s = torch.where(amax.isnan(), amax, (amax / (6.0 * g)).clamp(max=448.0)).to(torch.float8_e4m3fn)
        d = s.float() * g
    else:
        b = (amax / 6.0).view(torch.int32)
        code = ((b >> 23) + ((b & 0x7FFFFF) != 0).int()).clamp(max=254)
        code = torch.where(amax.isnan(), torch.full_like(code, 255), code).to(torch.uint8)
        s = code.view(torch.float8_e8m0fnu)
        d = torch.where(code == 255, torch.full_like(amax, float("nan")), torch.exp2(code.double() - 127).float())
    y = torch.where((d > 0)[..., None], v / d[..., None], torch.zeros_like(v))
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), s


def _values(q: torch.Tensor, s: torch.Tensor, gs: Optional[torch.Tensor]) -> torch.Tensor:
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1))
    v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], -1).flatten(-2)
    d = s.float()
    if gs is not None:
        d = d * (gs.reshape(-1, *([1] * (d.dim() - 1))) if gs.numel() > 1 else gs)
    return v * d.repeat_interleave(v.shape[-1] // max(1, s.shape[-1]), -1)


def dequantize_fp4_cpu(q, s, global_scale=None, dtype=None):
    block = _block_of(s, "s")
    _check(q.is_contiguous() and s.is_contiguous(), "q and s must be contiguous")
    _check_fp4(q, s, block, "dequantize_fp4:")
    _check_gscale(global_scale, block, _gscales_of(global_scale, q), "global_scale")
    dtype = torch.bfloat16 if dtype is None else dtype
    _check(dtype in (torch.bfloat16, torch.float16, torch.float32), "dtype must be bfloat16, float16 or float32")
    return _values(q, s, global_scale).to(dtype)


def _check_grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_gs, w_gs, n_step):
    for t, what in ((a_q, "a_q"), (a_s, "a_s"), (w_q, "w_q"), (w_s, "w_s"), (expert_offsets, "expert_offsets")):
        _check(t.is_contiguous(), f"{what} must be contiguous")
    block = _block_of(a_s, "a_s")
    _check(_block_of(w_s, "w_s") == block, "a_s and w_s must be of the same format")
    _check(a_q.dim() == 2 and w_q.dim() == 3 and a_q.shape[1] == w_q.shape[2], "a_q must be [M, K / 2] and w_q [E, N, K / 2]")
    k = _check_fp4(a_q, a_s, block, "a")
    _check_fp4(w_q, w_s, block, "w")
    _check(k % 128 == 0 and k > 0, f"K {k} must be a multiple of 128")
    _check(w_q.shape[1] % n_step == 0 and w_q.shape[1] > 0, f"N {w_q.shape[1]} must be a multiple of {n_step}")
    _check(expert_offsets.dtype == torch.int32 and expert_offsets.numel() == w_q.shape[0] + 1, "expert_offsets must be int32 [E+1]")
    _check_gscale(a_gs, block, 0, "a_global_scale")
    _check_gscale(w_gs, block, w_q.shape[0], "w_global_scale")
    return block


def _spans(expert_offsets: torch.Tensor, rows: int):
    """(expert, first row, last row + 1) of the experts that own rows; offsets outside [0, rows] are clamped."""
    off = [min(max(o, 0), rows) for o in expert_offsets.tolist()]
    return [(e, off[e], off[e + 1]) for e in range(len(off) - 1) if off[e] < off[e + 1]]


def _grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_gs, w_gs):
    out = torch.zeros(a_q.shape[0], w_q.shape[1])
    a = _values(a_q, a_s, a_gs)
    for e, lo, hi in _spans(expert_offsets, a_q.shape[0]):
        out[lo:hi] = a[lo:hi] @ _values(w_q[e], w_s[e], None if w_gs is None else w_gs[e]).t()
    return out


def grouped_gemm_fp4_cpu(a_q, a_s, w_q, w_s, expert_offsets, a_global_scale=None, w_global_scale=None):
    _check_grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_global_scale, w_global_scale, 128)
    return _grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_global_scale, w_global_scale).to(torch.bfloat16)


def grouped_gemm_fp4_swiglu_cpu(a_q, a_s, w_q, w_s, expert_offsets, a_global_scale=None, w_global_scale=None, out_global_scale=None):
    block = _check_grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_global_scale, w_global_scale, 256)
    _check_gscale(out_global_scale, block, 0, "out_global_scale")
    gate, up = _grouped_fp4(a_q, a_s, w_q, w_s, expert_offsets, a_global_scale, w_global_scale).chunk(2, -1)
    return quantize_fp4_cpu((torch.nn.functional.silu(gate) * up).contiguous(), block, out_global_scale)


def _check_mlp(x, w1, w2, expert_offsets):
    for t, what in ((x, "x"), (w1, "w1"), (w2, "w2"), (expert_offsets, "expert_offsets")):
        _check(t.is_contiguous(), f"{what} must be contiguous")
    _check(x.dtype in (torch.bfloat16, torch.float16), "grouped_mlp: x must be bfloat16 or float16")
    _check(w1.dtype == x.dtype and w2.dtype == x.dtype, "grouped_mlp: x, w1 and w2 must be of one type")
    _check(x.dim() == 2 and w1.dim() == 3 and w2.dim() == 3, "grouped_mlp: x must be [M, h], w1 [E, 2I, h], w2 [E, h, I]")
    h, e, i = x.shape[1], w1.shape[0], w2.shape[2]
    _check(tuple(w1.shape) == (e, 2 * i, h) and tuple(w2.shape) == (e, h, i), "grouped_mlp: x must be [M, h], w1 [E, 2I, h], w2 [E, h, I]")
    _check(h > 0 and i > 0 and h % 8 == 0 and i % 8 == 0, f"grouped_mlp: h {h} and I {i} must be multiples of 8")
    _check(expert_offsets.dtype == torch.int32 and expert_offsets.numel() == e + 1, "expert_offsets must be int32 [E+1]")


def grouped_mlp_train_cpu(x, w1, w2, expert_offsets):
    _check_mlp(x, w1, w2, expert_offsets)
    m, i = x.shape[0], w2.shape[2]
    y, act, gu = torch.zeros_like(x), torch.zeros(m, i, dtype=x.dtype), torch.zeros(m, 2 * i)
    for e, lo, hi in _spans(expert_offsets, m):
        gu[lo:hi] = x[lo:hi].float() @ w1[e].float().t()
        gate, up = gu[lo:hi].chunk(2, -1)
        act[lo:hi] = (torch.nn.functional.silu(gate) * up).to(x.dtype)
        y[lo:hi] = (act[lo:hi].float() @ w2[e].float().t()).to(x.dtype)
    return y, act, gu


def grouped_mlp_cpu(x, w1, w2, expert_offsets):
    return grouped_mlp_train_cpu(x, w1, w2, expert_offsets)[0]


def grouped_mlp_backward_cpu(dy, x, w1, w2, expert_offsets, act, gate_up, need_dx=True, need_dw1=True, need_dw2=True):
    _check_mlp(x, w1, w2, expert_offsets)
    _check(dy.dtype == x.dtype and dy.shape == x.shape and dy.is_contiguous(), "grouped_mlp: dy must be like x")
    _check(act.dtype == x.dtype and tuple(act.shape) == (x.shape[0], w2.shape[2]), "grouped_mlp: act must be [M, I]")
    _check(gate_up.dtype == torch.float32 and tuple(gate_up.shape) == (x.shape[0], 2 * w2.shape[2]), "grouped_mlp: gate_up must be float32 [M, 2I]")
    dx, dw1, dw2 = (torch.zeros_like(t) if need else t.new_empty(0) for t, need in ((x, need_dx), (w1, need_dw1), (w2, need_dw2)))
    for e, lo, hi in _spans(expert_offsets, x.shape[0]):
        g, u = gate_up[lo:hi].chunk(2, -1)
        d = dy[lo:hi].float()
        da, s = d @ w2[e].float(), torch.sigmoid(g)
        dgu = torch.cat([da * u * s * (1 + g * (1 - s)), da * g * s], -1).to(x.dtype).float()
        if need_dx:
            dx[lo:hi] = (dgu @ w1[e].float()).to(x.dtype)
        if need_dw1:
            dw1[e] = (dgu.t() @ x[lo:hi].float()).to(x.dtype)
        if need_dw2:
            dw2[e] = (d.t() @ act[lo:hi].float()).to(x.dtype)
    return dx, dw1, dw2


CPU_IMPLS = {
    "quantize_fp4": quantize_fp4_cpu,
    "dequantize_fp4": dequantize_fp4_cpu,
    "grouped_gemm_fp4": grouped_gemm_fp4_cpu,
    "grouped_gemm_fp4_swiglu": grouped_gemm_fp4_swiglu_cpu,
    "grouped_mlp": grouped_mlp_cpu,
    "grouped_mlp_train": grouped_mlp_train_cpu,
    "grouped_mlp_backward": grouped_mlp_backward_cpu,
}
