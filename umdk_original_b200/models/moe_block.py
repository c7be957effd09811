"""A pre-norm MoE block whose experts all live on this rank: residual and norm, routing, rows to the experts and back.

``FusedMoE`` is the layer of a group of ranks (8-bit weights, no gradient).  These classes need no ``Buffer``: ``MoEBlock`` trains
(16-bit experts, gradients of every parameter and of the input), ``Fp8MoEBlock`` serves the same block in 8 bits.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import ops
from .configs import MoEConfig
from .expert_mlp import ExpertMLP
from .weights import ExpertWeights, quantize_fp8_block


@dataclass(frozen=True)
class Routing:
    """How a block chooses experts (``ops.moe_route``).  ``group_top``: what a group of experts is worth, its best score or the sum of its
    two best."""
    topk: int
    score: str = "softmax"
    num_groups: int = 1
    topk_groups: int = 1
    group_top: int = 1
    renormalize: bool = True
    scale: float = 1.0

    def __call__(self, logits: torch.Tensor, bias: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
        return ops.moe_route(logits, self.topk, bias, self.score, self.num_groups, self.topk_groups, self.group_top, self.renormalize, self.scale)

    @staticmethod
    def of(cfg: MoEConfig, score: str = "softmax", scale: float = 1.0) -> "Routing":
        return Routing(cfg.topk, score, cfg.num_groups, cfg.topk_groups, 2 if score == "sigmoid" else 1, True, scale)


class MoEBlock(torch.nn.Module):
    """``s = x + residual``, ``y = norm(s)``, then the experts that the gate chooses for ``y``; trainable.

    With sigmoid scores ``route_bias`` (a buffer of zeros that a training loop may move to balance the experts) takes part in the
    choice and not in the weights."""

    def __init__(self, cfg: MoEConfig, dtype: torch.dtype = torch.bfloat16, device="cpu", seed: int = 0, score: str = "softmax", scale: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        g = torch.Generator(device=device)
        g.manual_seed(seed + 17)
        self.routing, self.eps = Routing.of(cfg, score, scale), eps
        self.norm_weight = torch.nn.Parameter(torch.ones(cfg.hidden, dtype=dtype, device=device))
        self.gate_weight = torch.nn.Parameter((torch.randn(cfg.num_experts, cfg.hidden, device=device, generator=g) * cfg.hidden ** -0.5).to(dtype))
        self.register_buffer("route_bias", torch.zeros(cfg.num_experts, device=device) if score == "sigmoid" else None)
        self.experts = ExpertMLP(cfg.num_experts, cfg.hidden, cfg.intermediate, dtype, device, seed)

    def _apply(self, fn, recurse=True):
        # a change of the block's type leaves the bias in fp32: the router takes no other, and its small steps would be lost in 16 bits
        bias = self.route_bias
        super()._apply(fn, recurse)
        if bias is not None and self.route_bias.dtype != bias.dtype:
            self.route_bias = bias.to(self.route_bias.device)
        return self

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """x [T, h], residual [T, h] (or None) -> (what the experts add [T, h], the residual stream after ``x`` [T, h]).  The next block
        takes both as they are."""
        if residual is None:
            y, total = ops.rms_norm(x, self.norm_weight, self.eps), x
        else:
            y, total = ops.add_rms_norm(x, residual, self.norm_weight, self.eps)
        # logits of y's type: the product's fp32 sums rounded once, so that the gate reads the rows as they are; equal ones go to the lowest expert
        idx, weights = self.routing(y @ self.gate_weight.t(), self.route_bias)
        rows, _, offsets, slots = ops.moe_group_rows(y, idx, self.gate_weight.shape[0])
        return ops.moe_ungroup_rows(self.experts(rows, offsets), slots, weights), total

    def quantized(self) -> "Fp8MoEBlock":
        """The block as it is now: training it further leaves the copy alone."""
        w = ExpertWeights(*quantize_fp8_block(self.experts.w1.detach()), *quantize_fp8_block(self.experts.w2.detach()))
        bias = None if self.route_bias is None else self.route_bias.clone()
        return Fp8MoEBlock(self.routing, self.norm_weight.detach().clone(), self.gate_weight.detach().clone(), bias, w, self.eps)


@dataclass
class Fp8MoEBlock:
    """The block for serving: rows leave the norm in e4m3 with power-of-two scales (and in 16 bits for the gate), travel to the experts
    in 8 bits and meet e4m3 weights there.  Hidden size and intermediate size are multiples of 128.  Plain tensors, no module."""
    routing: Routing
    norm_weight: torch.Tensor
    gate_weight: torch.Tensor
    route_bias: Optional[torch.Tensor]
    weights: ExpertWeights
    eps: float = 1e-6

    def __call__(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """As ``MoEBlock.forward``; what the experts add is bf16."""
        w = self.weights
        q, q_scales, total, y = ops.rms_norm_quant(x, self.norm_weight, 4, residual, self.eps, True)
        idx, weights = self.routing(y @ self.gate_weight.t(), self.route_bias)
        rows, scales, offsets, slots = ops.moe_group_rows(q, idx, self.gate_weight.shape[0], q_scales)
        act, act_scales = ops.grouped_gemm_fp8_swiglu(rows, scales, w.w1, w.s1, offsets, True)
        out = ops.grouped_gemm_fp8(act, act_scales, w.w2, w.s2, offsets, True)
        return ops.moe_ungroup_rows(out, slots, weights), x if residual is None else total
