"""grouped_mlp under PyTorch's transforms: compiled programs, forward mode, functorch.  CPU key unless marked."""
import numpy as np
import pytest
import torch

from fp4_cases import offsets_of
from umdk_original_b200 import ops
from umdk_original_b200.ops import cam_ops

pytestmark = pytest.mark.skipif(not cam_ops.native_loaded(), reason="native extension not built")


def tensors(dtype=torch.bfloat16, device="cpu", h=24, inter=16, rows=13, e=3):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(rows, h, generator=gen).to(dtype)
    w1 = (torch.randn(e, 2 * inter, h, generator=gen) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, inter, generator=gen) * inter ** -0.5).to(dtype)
    dy = torch.randn(rows, h, generator=gen).to(dtype)
    return [t.to(device) for t in (x, w1, w2, dy)]


def foreign(t):
    """The same values in memory that PyTorch does not own (as a dispatch hands out), and the memory as bytes."""
    mem = np.empty(t.numel() * t.element_size(), dtype=np.uint8)
    view = torch.from_numpy(mem).view(t.dtype).view(t.shape)
    view.copy_(t)
    return view, mem


@pytest.mark.parametrize("backend", ["eager", "aot_eager", "aot_eager_decomp_partition"])
def test_rows_overwritten_before_the_backward_pass(backend):
    """What a dispatch on the same Buffer does to rows and offsets between the passes, behind autograd's back."""
    x, w1, w2, dy = tensors()
    off = offsets_of([4, 3, 6])
    w1.requires_grad_()
    w2.requires_grad_()
    want = torch.autograd.grad(ops.grouped_mlp(x, w1, w2, off), (w1, w2), dy)
    fn = torch.compile(lambda *a: ops.grouped_mlp(*a), backend=backend, fullgraph=True)
    (fx, mx), (fo, mo) = foreign(x), foreign(off)
    y = fn(fx, w1, w2, fo)
    mx[:], mo[:] = 0, 0
    got = torch.autograd.grad(y, (w1, w2), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("backend", ["aot_eager", "aot_eager_decomp_partition"])
def test_compiled_is_eager(backend):
    x, w1, w2, dy = tensors()
    off = offsets_of([4, 0, 6], head=1)
    runs = []
    for fn in (ops.grouped_mlp, torch.compile(lambda *a: ops.grouped_mlp(*a), backend=backend, fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
        y = fn(*leaves, off)
        runs.append((y.detach(), *torch.autograd.grad(y, leaves, dy), fn(x, w1, w2, off)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(which, no_grad):
    """A tangent is not dropped: neither by dual tensors nor by torch.func.jvp, whichever operand carries it."""
    import torch.autograd.forward_ad as fwad
    args = tensors()[:3]
    off = offsets_of([4, 3, 6])

    def f(t):
        return ops.grouped_mlp(*[t if i == which else a for i, a in enumerate(args)], off)
    with torch.set_grad_enabled(not no_grad):
        with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            f(fwad.make_dual(args[which], torch.ones_like(args[which])))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(f, (args[which],), (torch.ones_like(args[which]),))
        with fwad.dual_level():
            assert torch.equal(f(args[which]), f(args[which].clone()))  # nothing here carries a tangent


def test_functorch():
    """Batches of calls are computed one by one; gradients inside torch.func are refused, not left out."""
    x, w1, w2, dy = tensors()
    off = offsets_of([4, 3, 6])
    xs = torch.stack([x, x.flip(0)])
    got = torch.func.vmap(lambda t: ops.grouped_mlp(t, w1, w2, off))(xs)
    assert torch.equal(got, torch.stack([ops.grouped_mlp(t, w1, w2, off) for t in xs]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda w: ops.grouped_mlp(x, w, w2, off).float().sum())(w1)


@pytest.mark.gpu
def test_compiled_layers_after_the_next_dispatch():
    """Two compiled layers share a Buffer: the second dispatch overwrites the rows that the first layer's experts saw."""
    from umdk_original_b200 import Buffer, CamConfig
    from umdk_original_b200.models import ExpertMLP, offsets_from_counts
    dev = torch.device("cuda", 0)
    t, h, inter, e, k = 32, 128, 64, 4, 2
    gen = torch.Generator().manual_seed(11)
    idx = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)]).to(dev)
    wt = torch.rand(t, k, generator=gen).to(dev)
    buf = Buffer(None, CamConfig(num_experts=e, max_tokens=t, hidden=h, topk=k, timeout_ms=2000.0), name="expert_mlp_compiled",
                 device=dev, rank=0, num_ranks=1)
    layers = [ExpertMLP(e, h, inter, device=dev, seed=s) for s in (1, 2)]
    loss, rows = 0.0, []
    for layer in layers:
        x = torch.randn(t, h, generator=gen).to(torch.bfloat16).to(dev)
        rx, _, _, per_e, _ = ops.moe_dispatch_prefill_quant(x, idx, wt, buf.capacity, buf.name, 0, 1, 0)
        off = offsets_from_counts(per_e)
        rows.append((rx, rx.clone(), off))
        loss = loss + torch.compile(layer, backend="aot_eager", fullgraph=True)(rx, off).float().square().sum()
    assert not torch.equal(rows[0][0], rows[0][1])  # overwritten
    got = torch.autograd.grad(loss, [p for layer in layers for p in (layer.w1, layer.w2)])
    want = []
    for layer, (_, rx, off) in zip(layers, rows):
        want += torch.autograd.grad(layer(rx, off).float().square().sum(), (layer.w1, layer.w2))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf.check()
    buf.destroy()
