"""The block that runs norm, routing, rows to the experts and back together: 16-bit experts with gradients, 8-bit ones."""
import dataclasses

import pytest
import torch

from umdk_original_b200 import ops
from umdk_original_b200.models import TINY, MoEBlock, MoEConfig
from umdk_original_b200.ops import cam_ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GROUPED = MoEConfig("grouped", 256, 128, 16, 4, 32, num_groups=4, topk_groups=2)
native = pytest.mark.skipif(not cam_ops.native_loaded(), reason="native extension not built")


def make(cfg, device, score="softmax", dtype=torch.bfloat16, tokens=40):
    block = MoEBlock(cfg, dtype, device, seed=3, score=score, scale=1.5)
    g = torch.Generator(device=device).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    with torch.no_grad():
        block.norm_weight.copy_(1 + 0.2 * r(cfg.hidden))
        if block.route_bias is not None:
            block.route_bias.copy_(0.05 * r(cfg.num_experts))
    return block, r(tokens, cfg.hidden).to(dtype), r(tokens, cfg.hidden).to(dtype), r(tokens, cfg.hidden).to(dtype), r(tokens, cfg.hidden).to(dtype)


def block64(block, x, residual, choice):
    """The block's formula in 64 bits on the choice that the block made, differentiable."""
    p = {n: t.detach().double().requires_grad_() for n, t in block.named_parameters()}
    a, b = x.double().requires_grad_(), residual.double().requires_grad_()
    s = a + b
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + block.eps) * p["norm_weight"]
    logits = y @ p["gate_weight"].t()
    score = torch.sigmoid(logits) if block.routing.score == "sigmoid" else torch.softmax(logits, -1)
    w = score.gather(1, choice)
    w = w / w.sum(-1, keepdim=True) * block.routing.scale
    gu = torch.einsum("th,eih->tei", y, p["experts.w1"])
    gate, up = gu.chunk(2, -1)
    z = torch.einsum("tei,ehi->teh", torch.nn.functional.silu(gate) * up, p["experts.w2"])
    picked = z.gather(1, choice[..., None].expand(-1, -1, z.shape[-1]))
    return (picked * w[..., None]).sum(1), s, p, a, b


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cfg,score", [(TINY, "softmax"), (GROUPED, "softmax"), (GROUPED, "sigmoid")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_and_gradients(device, cfg, score, dtype):
    block, x, res, dout, ds = make(cfg, device, score, dtype)
    leaves = [x.requires_grad_(), res.requires_grad_()]
    out, s = block(*leaves)
    params = dict(block.named_parameters())
    grads = torch.autograd.grad((out, s), [*leaves, *params.values()], (dout, ds))
    with torch.no_grad():
        y, s2 = ops.add_rms_norm(x, res, block.norm_weight, block.eps)
        idx, _ = block.routing(y @ block.gate_weight.t(), block.route_bias)
    out64, s64, p, a, b = block64(block, x.detach(), res.detach(), idx)
    want = torch.autograd.grad((out64, s64), [a, b, *p.values()], (dout.double(), ds.double()))
    # Every result is at most a dozen roundings of operands away from the inputs (sum, y, logits, act, z, out, and back dz, dact, dgu, rows, dy,
    # dx): each moves the vector by half a step, relative, and none of the maps between them stretches a random error more than the
    # signal.  The gate's gradient goes through differences of weights, where half of the signal may cancel.
    half = torch.finfo(dtype).eps / 2
    for name, got, ref in zip(["out", "sum", "x", "residual", *params], [out, s, *grads], [out64, s64, *want]):
        off = float((got.detach().double() - ref.detach()).norm() / ref.detach().norm())
        assert off <= (24 if name == "gate_weight" else 12) * half, (name, off / half)
    assert torch.equal(s2, s)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_block_in_8_bits(device, score):
    """Beside the 16-bit block: e4m3 rows and weights (half a step 2^-4 relative at most, 2^-5.8 on the mean), activations once more."""
    block, x, res, _, _ = make(GROUPED, device, score)
    fp8 = block.quantized()
    with torch.no_grad():
        out, s = fp8(x, res)
        want, s2 = block(x, res)
        first, alone = fp8(x)
        assert alone is x and first.shape == x.shape
    assert torch.equal(s, s2) and out.dtype == torch.bfloat16
    # rows, w1, activation, w2: four independent roundings, their rms 2^-5.8 each, the last two after a product of two
    off = float((out.double() - want.double()).norm() / want.double().norm())
    assert off <= 2.0 ** -4 * 2, off


@native
@pytest.mark.parametrize("device", DEVICES)
def test_two_blocks_in_a_row(device):
    """The stream goes from block to block as it is; gradients reach the first input."""
    block, x, _, dout, _ = make(TINY, device)
    x.requires_grad_()
    out, s = block(x)
    out, s = block(out, s)
    (out + s).backward(dout)
    assert x.grad.isfinite().all() and all(p.grad.isfinite().all() and p.grad.any() for p in block.parameters())


@pytest.mark.parametrize("device", DEVICES)
def test_block_without_tokens(device):
    block, x, res, _, _ = make(TINY, device)
    with torch.no_grad():
        out, s = block(x[:0], res[:0])
    assert out.shape == s.shape == (0, TINY.hidden)
    assert dataclasses.replace(block.routing, topk=1).topk == 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_8_bit_block_is_a_snapshot(device, score):
    """What is trained after it was taken does not reach it: not the norm and the router either."""
    block, x, res, _, _ = make(GROUPED, device, score)
    fp8 = block.quantized()
    with torch.no_grad():
        want = [t.clone() for t in fp8(x, res)]
        for t in (*block.parameters(), *block.buffers()):
            t.add_(0.5)
        assert all(torch.equal(a, b) for a, b in zip(fp8(x, res), want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_block_of_another_type(device, score):
    """A block that was made in one 16-bit type runs in the other; the selection bias stays as it is, in fp32, wherever the block goes."""
    block, x, res, _, _ = make(GROUPED, device, score, torch.float16)
    bias = None if block.route_bias is None else block.route_bias.clone()
    block = block.to(torch.bfloat16)
    with torch.no_grad():
        out, s = block(x.bfloat16(), res.bfloat16())
        assert out.dtype == s.dtype == torch.bfloat16 and block.quantized()(x.bfloat16(), res.bfloat16())[0].shape == out.shape
    assert bias is None if score == "softmax" else block.route_bias.dtype == torch.float32 and torch.equal(block.route_bias, bias)
    back = block.half().cpu()
    assert all(p.dtype == torch.float16 and p.device.type == "cpu" for p in back.parameters())
    assert bias is None or torch.equal(back.state_dict()["route_bias"], bias.cpu())
