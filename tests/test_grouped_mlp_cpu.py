"""Gated feed-forward block of 16-bit experts and the expert modules on the CPU key: values, gradients, refusals."""
import pytest
import torch

from fp4_cases import offsets_of
from umdk_original_b200 import ops
from umdk_original_b200.models import ExpertMLP, Fp4ExpertMLP


def block64(x, w1, w2, off):
    """The formula in fp64, differentiable."""
    parts = [x.new_zeros(off[0], x.shape[1])]
    for e in range(w1.shape[0]):
        g, u = (x[off[e]: off[e + 1]] @ w1[e].T).chunk(2, -1)
        parts.append((g * torch.sigmoid(g) * u) @ w2[e].T)
    parts.append(x.new_zeros(x.shape[0] - off[-1], x.shape[1]))
    return torch.cat(parts)


def tensors(dtype, device="cpu", h=24, inter=16, rows=13, e=3):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(rows, h, generator=gen).to(dtype)
    w1 = (torch.randn(e, 2 * inter, h, generator=gen) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, inter, generator=gen) * inter ** -0.5).to(dtype)
    dy = torch.randn(rows, h, generator=gen).to(dtype)
    return [t.to(device) for t in (x, w1, w2, dy)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_and_gradients(dtype):
    x, w1, w2, dy = tensors(dtype)
    off = offsets_of([4, 0, 6], head=1)
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    got = torch.autograd.grad(y, leaves, dy)
    l64 = [t.double().requires_grad_() for t in (x, w1, w2)]
    y64 = block64(*l64, off.tolist())
    want = torch.autograd.grad(y64, l64, dy.double())
    # three roundings at most (act or dgu, the result, and subnormals of fp16) of at most half a step each, sums of a few dozen
    # terms of order 1 that enter with both signs: 4 half steps of the largest magnitude
    half = torch.finfo(dtype).eps / 2
    for a, b in zip((y, *got), (y64, *want)):
        assert a.dtype == dtype
        assert (a.double() - b).abs().max() <= 4 * half * b.abs().max() + 1e-6
    assert (y[0] == 0).all() and (y[11:] == 0).all() and (got[1][1] == 0).all()


def test_gradients_against_differences():
    """The formula of the gradients against central differences of the formula in fp64."""
    x, w1, w2, _ = tensors(torch.float64, rows=6, h=8, inter=8, e=2)
    off = [0, 4, 6]
    assert torch.autograd.gradcheck(lambda a, b, c: block64(a, b, c, off), [t.requires_grad_() for t in (x, w1, w2)])


@pytest.mark.parametrize("which", range(3))
def test_only_wanted_gradients(which):
    x, w1, w2, dy = tensors(torch.bfloat16)
    off = offsets_of([4, 3, 6])
    full = [t.clone().requires_grad_() for t in (x, w1, w2)]
    want = torch.autograd.grad(ops.grouped_mlp(*full, off), full, dy)[which]
    part = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, w1, w2))]
    got, = torch.autograd.grad(ops.grouped_mlp(*part, off), part[which], dy)
    assert torch.equal(got, want)
    part = ops.grouped_mlp_backward(dy, x, w1, w2, off, *ops.grouped_mlp_train(x, w1, w2, off)[1:], which == 0, which == 1, which == 2)
    assert torch.equal(part[which], want) and all(t.numel() == 0 for i, t in enumerate(part) if i != which)


def test_broadcast_gradient_and_no_second_derivative():
    x, w1, w2, _ = tensors(torch.bfloat16)
    off = offsets_of([4, 3, 6])
    leaf = x.clone().requires_grad_()
    y = ops.grouped_mlp(leaf, w1, w2, off)
    got, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)  # the gradient of a sum is an expanded scalar
    want, = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(), create_graph=True)
        torch.autograd.grad(g.sum(), leaf)


def test_empty_and_meta():
    x, w1, w2, dy = tensors(torch.bfloat16)
    off = offsets_of([0, 0, 0])
    leaves = [t.clone().requires_grad_() for t in (x[:0], w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    dx, dw1, dw2 = torch.autograd.grad(y, leaves, dy[:0])
    assert y.shape == (0, 24) and dx.shape == (0, 24) and (dw1 == 0).all() and (dw2 == 0).all()
    m = [t.to("meta") for t in (x, w1, w2, off)]
    assert ops.grouped_mlp(*m).shape == x.shape
    y, act, gu = ops.grouped_mlp_train(*m)
    assert act.shape == (13, 16) and gu.shape == (13, 32) and gu.dtype == torch.float32


def refusals(device):
    x, w1, w2, dy = tensors(torch.bfloat16, device)
    off = offsets_of([4, 3, 6], device=device)
    y, act, gu = ops.grouped_mlp_train(x, w1, w2, off)
    odd = tensors(torch.bfloat16, device, h=20)
    f = ops.grouped_mlp
    return [
        lambda: f(x.float(), w1.float(), w2.float(), off),
        lambda: f(x.half(), w1, w2, off),
        lambda: f(x[:, :16], w1, w2, off),
        lambda: f(x.t().contiguous().t(), w1, w2, off),
        lambda: f(x, w1[:, :-2].contiguous(), w2, off),
        lambda: f(x, w1, w2[:2].contiguous(), off),
        lambda: f(x, w1, w2, off[:-1].contiguous()),
        lambda: f(x, w1, w2, off.long()),
        lambda: f(x[0], w1, w2, off),
        lambda: f(odd[0], odd[1], odd[2], off),
        lambda: ops.grouped_mlp_backward(dy.float(), x, w1, w2, off, act, gu),
        lambda: ops.grouped_mlp_backward(dy, x, w1, w2, off, act[:, :8].contiguous(), gu),
        lambda: ops.grouped_mlp_backward(dy, x, w1, w2, off, act, gu.bfloat16()),
    ]


@pytest.mark.parametrize("i", range(13))
def test_refusals(i):
    with pytest.raises(RuntimeError, match="umdk_cam_op_lib"):
        refusals("cpu")[i]()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantised_module(fmt):
    """4-bit experts stay near the experts they come from: e2m1 rounds a value by an eighth of it at most between its points (and
    by half of the smallest step below), three operands do."""
    m = ExpertMLP(2, 128, 128, seed=3)
    x = torch.randn(9, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    off = offsets_of([5, 4])
    q = m.quantized(fmt)
    want = m(x, off).float()
    err = (q(x, off).float() - want).norm() / want.norm()
    assert err < 0.35 and q.nbytes() < 0.3 * sum(p.numel() * 2 for p in m.parameters())
    with pytest.raises(ValueError):
        m.quantized("int4")
