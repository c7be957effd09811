"""Local experts as modules that take the rows a dispatch delivered: unquantised and trainable, or in 4 bits.

``moe_dispatch_prefill`` and ``moe_dispatch_shmem`` with ``quantMode`` 0 hand out bf16 (fp16) rows grouped by local expert;
these classes run the expert MLP on them, and ``moe_combine_prefill`` / ``moe_combine_shmem`` take the result.  The fused layer
(``FusedMoE``) stays the route for fp8 and int8 weights.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .. import ops


def offsets_from_counts(rows_per_expert: torch.Tensor) -> torch.Tensor:
    """int32 [E_l + 1]: first row of every expert and the end of the last, from rows per expert; on their device, no host read."""
    return torch.cat([rows_per_expert.new_zeros(1), rows_per_expert.cumsum(0)]).to(torch.int32)


class ExpertMLP(torch.nn.Module):
    """``w2 (silu(w1_gate x) * w1_up x)`` of every local expert in bf16 or fp16, with its backward pass (``ops.grouped_mlp``).

    ``w1 [E_l, 2I, h]`` (gate rows first) and ``w2 [E_l, h, I]`` are the layouts of ``ExpertWeights``."""

    def __init__(self, num_local: int, hidden: int, inter: int, dtype: torch.dtype = torch.bfloat16, device="cpu", seed: int = 0):
        super().__init__()
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.w1 = torch.nn.Parameter((torch.randn(num_local, 2 * inter, hidden, device=device, generator=g) * hidden ** -0.5).to(dtype))
        self.w2 = torch.nn.Parameter((torch.randn(num_local, hidden, inter, device=device, generator=g) * inter ** -0.5).to(dtype))

    def forward(self, rows: torch.Tensor, expert_offsets: torch.Tensor) -> torch.Tensor:
        """rows [M, h], expert_offsets int32 [E_l + 1] (``offsets_from_counts`` of what the dispatch returns) -> [M, h]; rows of no
        expert give zeros."""
        return ops.grouped_mlp(rows, self.w1, self.w2, expert_offsets)

    def quantized(self, fmt: str = "nvfp4") -> "Fp4ExpertMLP":
        return Fp4ExpertMLP.from_dense(self.w1.detach(), self.w2.detach(), fmt)


@dataclass
class Fp4ExpertMLP:
    """The same experts in 4 bits: ``nvfp4`` (e4m3 scale per 16 values and one fp32 scale per expert) or ``mxfp4`` (power-of-two
    scale per 32).  Rows are quantised on the way in, the activation between the two products is quantised by the first one.

    nvfp4 block scales reach from 2^-9 to 448.  With ``x_gs`` and ``act_gs`` at None (1) rows and activations have to fit them: blocks
    whose largest magnitude is below 6 x 2^-10 become zeros, what is above 2688 is cut; ``calibrate`` sets both from sample rows.
    mxfp4 scales reach over the whole range of fp32.  Plain tensors, no module: move or store the fields."""
    w1_q: torch.Tensor   # [E_l, 2I, h / 2] e2m1 pairs
    w1_s: torch.Tensor   # [E_l, 2I, h / block]
    w2_q: torch.Tensor   # [E_l, h, I / 2]
    w2_s: torch.Tensor   # [E_l, h, I / block]
    w1_gs: Optional[torch.Tensor] = None   # nvfp4: [E_l] fp32
    w2_gs: Optional[torch.Tensor] = None
    x_gs: Optional[torch.Tensor] = None    # nvfp4: [1] fp32, scales of the rows and of the activation (a calibration's result);
    act_gs: Optional[torch.Tensor] = None  # None stands for 1

    @property
    def block(self) -> int:
        return 16 if self.w1_s.dtype == torch.float8_e4m3fn else 32

    @staticmethod
    def from_dense(w1: torch.Tensor, w2: torch.Tensor, fmt: str = "nvfp4") -> "Fp4ExpertMLP":
        if fmt not in ("nvfp4", "mxfp4"):
            raise ValueError(f"format {fmt!r}: nvfp4 or mxfp4")
        if fmt == "mxfp4":
            return Fp4ExpertMLP(*ops.quantize_fp4(w1, 32), *ops.quantize_fp4(w2, 32))

        def one(w):
            # the largest block scale of an expert becomes 448, the largest e4m3; an expert of zeros keeps 1
            top = w.flatten(1).abs().amax(1).float()
            gs = torch.where(top > 0, top / (6.0 * 448.0), torch.ones_like(top))
            return (*ops.quantize_fp4(w, 16, gs), gs)
        q1, s1, g1 = one(w1)
        q2, s2, g2 = one(w2)
        return Fp4ExpertMLP(q1, s1, q2, s2, g1, g2)

    @torch.no_grad()
    def calibrate(self, rows: torch.Tensor, expert_offsets: torch.Tensor, margin: float = 4.0) -> "Fp4ExpertMLP":
        """nvfp4: sets ``x_gs`` and ``act_gs`` so that the largest row value and the largest activation that these rows give have block
        scales of 448 / ``margin``: later ones may be ``margin`` times as large, and 1000 times smaller without losing bits of
        their scales.  Rows of no expert do not count.  Waits for the device; nothing to do for mxfp4."""
        if self.block == 32:
            return self

        def scale(values: torch.Tensor, what: str) -> torch.Tensor:
            top = float(values.abs().amax()) if values.numel() else 0.0
            if not top < float("inf"):
                raise ValueError(f"calibrate: {what} hold NaN or infinity")
            return torch.full((1,), top * margin / (6.0 * 448.0) if top > 0 else 1.0, dtype=torch.float32, device=rows.device)
        first, last = (min(max(int(expert_offsets[i]), 0), rows.shape[0]) for i in (0, -1))
        self.x_gs = scale(rows[first:last].float(), "rows")
        q, s = ops.quantize_fp4(rows, 16, self.x_gs)
        gate, up = ops.grouped_gemm_fp4(q, s, self.w1_q, self.w1_s, expert_offsets, self.x_gs, self.w1_gs)[first:last].float().chunk(2, -1)
        self.act_gs = scale(torch.nn.functional.silu(gate) * up, "activations")
        return self

    def __call__(self, rows: torch.Tensor, expert_offsets: torch.Tensor) -> torch.Tensor:
        """rows [M, h] bf16 / fp16 / fp32 -> [M, h] bf16; rows of no expert give zeros."""
        q, s = ops.quantize_fp4(rows, self.block, self.x_gs)
        q, s = ops.grouped_gemm_fp4_swiglu(q, s, self.w1_q, self.w1_s, expert_offsets, self.x_gs, self.w1_gs, self.act_gs)
        return ops.grouped_gemm_fp4(q, s, self.w2_q, self.w2_s, expert_offsets, self.act_gs, self.w2_gs)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.w1_q, self.w1_s, self.w2_q, self.w2_s, self.w1_gs, self.w2_gs) if t is not None)
