"""Expert-MLP operators that need no ``Buffer``: schemas and CPU implementations.

``quantize_fp4`` / ``dequantize_fp4`` / ``grouped_gemm_fp4`` / ``grouped_gemm_fp4_swiglu``: 4-bit floating point with block
scales (the formats are described in csrc/common/fp4.cuh).  The CUDA implementations live in csrc/bindings_expert.cpp; the CPU
ones here follow the same contracts in fp32, expert by expert.
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


CPU_IMPLS = {
    "quantize_fp4": quantize_fp4_cpu,
    "dequantize_fp4": dequantize_fp4_cpu,
    "grouped_gemm_fp4": grouped_gemm_fp4_cpu,
    "grouped_gemm_fp4_swiglu": grouped_gemm_fp4_swiglu_cpu,
}
