"""Norm, routing and rows grouped by expert against their definitions in 64 bits: the CPU implementations here, the kernels on a B200."""
import gc
import weakref

import pytest
import torch

from layer_cases import (U, group64, half_step, norm64, norm_grad_tol, norm_grads64, norm_tol, route64, route_grad64, route_weight_tol, weight_grad_tol,
                         within)
from umdk_original_b200 import ops
from umdk_original_b200.ops import cam_ops, reference as ref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
BF, HF, FL = DTYPES
native = pytest.mark.skipif(not cam_ops.native_loaded(), reason="native extension not built")


def gen(device, seed=0):
    return torch.Generator(device=device).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------
# Norm
# ------------------------------------------------------------------------------------------------
# widths on both sides of the kernels' borders: 512 and 1024 (a warp with one or two sixteens, a block), 8192 (blocks of 512 threads
# backward), and of multiples of 8 and 16
WIDTHS = [1, 7, 8, 64, 255, 256, 264, 512, 520, 1000, 1024, 1032, 1023, 2056, 4096, 7168, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,residual,weight", [(BF, None, BF), (BF, BF, BF), (BF, FL, FL), (HF, HF, HF), (HF, FL, HF), (FL, FL, FL), (FL, None, FL), (HF, None, FL)])
@pytest.mark.parametrize("h", WIDTHS)
def test_norm_and_gradients(device, dtype, residual, weight, h):
    g = gen(device, h)
    rows, eps = (11, 1e-6) if h > 512 else (37, 1e-5)
    x = randn(g, rows, h, dtype=dtype, scale=3.0)
    r = None if residual is None else randn(g, rows, h, dtype=residual)
    w = randn(g, h, dtype=weight)
    y64, total64, _ = norm64(x, r, w, eps)
    with torch.no_grad():
        got = (ops.rms_norm(x, w, eps), None) if r is None else ops.add_rms_norm(x, r, w, eps)
    assert got[0].dtype == dtype
    within(got[0], y64, norm_tol(y64, dtype), "y")
    if r is not None:
        assert got[1].dtype == residual and torch.equal(got[1], total64)
    if not cam_ops.native_loaded():
        return
    leaves = [t.clone().requires_grad_() for t in (x, r, w) if t is not None]
    out = (ops.rms_norm(leaves[0], leaves[1], eps),) if r is None else ops.add_rms_norm(*leaves, eps)
    assert torch.equal(out[0], got[0])
    dy = randn(g, rows, h, dtype=dtype)
    ds = None if r is None else randn(g, rows, h, dtype=residual)
    grads = torch.autograd.grad(out, leaves, [t for t in (dy, ds) if t is not None])
    d, size, dw, dw_size = norm_grads64(dy, ds, total64, w, eps)
    within(grads[0], d, norm_grad_tol(d, size, dtype), "dx")
    if r is not None:
        assert grads[1].dtype == residual
        within(grads[1], d, norm_grad_tol(d, size, residual), "dresidual")
    within(grads[-1], dw, weight_grad_tol(dw, dw_size, rows, weight), "dweight")


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,h", [(1, 4096), (5000, 72), (2400, 520), (701, 1000)])
def test_norm_weight_gradient_of_many_rows(device, rows, h):
    """More rows than blocks: every block goes round several times."""
    g = gen(device, rows)
    x, w, dy = randn(g, rows, h, dtype=BF), randn(g, h, dtype=FL), randn(g, rows, h, dtype=BF)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    dx, dweight = torch.autograd.grad(ops.rms_norm(*leaves), leaves, dy)
    d, size, dw, dw_size = norm_grads64(dy, None, x.detach(), w.detach(), 1e-6)
    within(dx, d, norm_grad_tol(d, size, BF), "dx")
    within(dweight, dw, weight_grad_tol(dw, dw_size, rows, FL), "dweight")
    assert torch.equal(dweight, torch.autograd.grad(ops.rms_norm(*leaves), leaves, dy)[1])  # the same bits again


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,residual", [(BF, BF), (HF, FL)])
def test_norm_gradients_of_one_output_or_one_input(device, dtype, residual):
    """Gradients that are not asked for are left out, outputs without a gradient count as zeros."""
    g = gen(device, 3)
    x, r, w = randn(g, 5, 264, dtype=dtype), randn(g, 5, 264, dtype=residual), randn(g, 264, dtype=dtype)
    dy, ds = randn(g, 5, 264, dtype=dtype), randn(g, 5, 264, dtype=residual)
    all_ = [t.clone().requires_grad_() for t in (x, r, w)]
    both = torch.autograd.grad(ops.add_rms_norm(*all_), all_, (dy, ds))
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, r, w))]
        (got,) = torch.autograd.grad(ops.add_rms_norm(*args), args[i], (dy, ds))
        assert torch.equal(got, both[i])
    only_y = torch.autograd.grad(ops.add_rms_norm(*all_)[0], all_, dy)
    zeros = torch.autograd.grad(ops.add_rms_norm(*all_), all_, (dy, torch.zeros_like(ds)))
    assert all(torch.equal(a, b) for a, b in zip(only_y, zeros))
    only_s = torch.autograd.grad(ops.add_rms_norm(*all_)[1], all_, ds, allow_unused=True)
    assert torch.equal(only_s[0], ds.to(dtype)) and torch.equal(only_s[1], ds) and not only_s[2].any()


@native
@pytest.mark.parametrize("device", DEVICES)
def test_norm_gradients_against_differences(device):
    """Central differences in fp32: (f(x + a v) - f(x - a v)) / 2a against the gradient along v."""
    g = gen(device, 4)
    x, r, w = (randn(g, *s).requires_grad_() for s in ((3, 40), (3, 40), (40,)))
    dy, ds = randn(g, 3, 40), randn(g, 3, 40)
    grads = torch.autograd.grad(ops.add_rms_norm(x, r, w), (x, r, w), (dy, ds))

    def f(*args):
        y, s = ops.add_rms_norm(*args)
        return float((y.double() * dy.double()).sum() + (s.double() * ds.double()).sum())
    with torch.no_grad():
        for i, t in enumerate((x, r, w)):
            v, a = randn(g, *t.shape), 2.0 ** -7
            args = [x, r, w]
            hi, lo = [[*args[:i], t + sign * a * v, *args[i + 1:]] for sign in (1, -1)]
            want = float((grads[i].double() * v.double()).sum())
            # differences: third derivatives (a^2) and roundings of 240 terms of a few units each over 2 a
            assert abs((f(*hi) - f(*lo)) / (2 * a) - want) <= 2.0 ** -7 * (1 + abs(want))


@pytest.mark.parametrize("device", DEVICES)
def test_norm_special_rows(device):
    x = torch.zeros(6, 264, dtype=BF, device=device)
    w = torch.ones(264, dtype=BF, device=device)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    x[3] = 1e-20
    x[4] = 3e4
    y = ops.rms_norm(x, w)
    assert not y[0].any() and y[1].isnan().all() and not y[5].any()
    assert y[2, 7].isnan() and not y[2, :7].any()  # 1 / rms is zero
    assert torch.equal(y[4], torch.ones_like(y[4]))
    assert torch.equal(y[3], (x[3].float() * 1e3).to(BF))  # eps alone
    q, s, _, _ = ops.rms_norm_quant(x, w, 2)
    assert s[1].isnan() and not q[0].any() and q[4].eq(127).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,residual", [(BF, None), (BF, BF), (HF, FL), (FL, FL), (FL, None)])
@pytest.mark.parametrize("mode,h", [(2, 8), (2, 77), (2, 1000), (2, 4096), (2, 16384), (2, 9001), (3, 128), (3, 384), (3, 1024), (3, 1152), (3, 7168),
                                    (4, 128), (4, 640), (4, 4096), (4, 8192), (4, 8320), (4, 16384)])
def test_norm_quant(device, dtype, residual, mode, h):
    g = gen(device, h + mode)
    rows = 9
    x = randn(g, rows, h, dtype=dtype) * torch.exp(randn(g, h)).to(dtype)
    r = None if residual is None else randn(g, rows, h, dtype=residual)
    w = randn(g, h, dtype=dtype)
    y64, total64, _ = norm64(x, r, w, 1e-6)
    q, s, total, y = ops.rms_norm_quant(x, w, mode, r, 1e-6, True)
    bare = ops.rms_norm_quant(x, w, mode, r, 1e-6)
    assert torch.equal(bare[0].view(torch.int8), q.view(torch.int8)) and torch.equal(bare[1], s) and bare[3].numel() == 0
    within(y, y64, norm_tol(y64, dtype), "rows")
    assert torch.equal(total, total64) if r is not None else total.numel() == 0
    rel = 40 * U  # of a value of y (32 u), a scale's division and product
    if mode == 2:
        assert q.dtype == torch.int8 and tuple(s.shape) == (rows,)
        want = y64.abs().amax(-1) / 127
        within(s, want, want * rel, "scales")
        # half a step of the row's scale
        within(q.double() * s.double()[:, None], y64, s.double()[:, None] * (0.5 + 127 * 3 * rel), "values")
        return
    assert q.dtype == torch.float8_e4m3fn and tuple(s.shape) == (rows, h // 128)
    want = y64.view(rows, -1, 128).abs().amax(-1).clamp(min=1e-4) / 448
    if mode == 3:
        within(s, want, want * rel, "scales")
    else:
        assert torch.equal(torch.exp2(torch.log2(s.double()).round()), s.double())
        assert (s.double() >= want * (1 - rel)).all() and (s.double() < 2 * want * (1 + rel)).all()
    v = y64 / s.double().repeat_interleave(128, -1)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)  # 2^-9 at the least
    within(q, v.clamp(-448, 448), step / 2 + v.abs() * 3 * rel, "codes")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mode", [2, 3, 4])
@pytest.mark.parametrize("h", [128, 1024, 7168])
def test_norm_quant_is_that_of_the_dispatch(device, mode, h):
    """fp32 rows come out as they were quantised: codes and scales are the bits that the dispatch's formula has for them, up to 3e38."""
    g = gen(device, h)
    x, w = randn(g, 64, h), randn(g, h)
    w[1] = 5e37
    for weight in (w[2:3].expand(h).contiguous(), w):
        q, s, _, y = (t.cpu() for t in ops.rms_norm_quant(x, weight, mode, None, 1e-6, True))
        q2, s2 = ref.quant_int8_token(y) if mode == 2 else ref.quant_fp8_1x128(y, mode == 4)
        assert y.isfinite().all() and torch.equal(s.view(s2.shape), s2) and torch.equal(q.float(), q2.float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("mode", [3, 4])
@pytest.mark.parametrize("h", [128, 1152, 7168])
def test_norm_e4m3_rows_that_are_not_finite(device, dtype, mode, h):
    """NaN behind the norm: its block has a NaN scale and NaN codes.  An infinity: an infinite scale, a NaN code, zeros beside it.  Other
    blocks and rows are as without."""
    g = gen(device, h)
    x, w = randn(g, 5, h, dtype=dtype), torch.rand(h, generator=g, device=device) + 0.5
    want_q, want_s = (t.float() for t in ops.rms_norm_quant(x, w, mode)[:2])
    n, at = h // 128 - 1, torch.arange(h, device=device) == h - 3
    for value in (float("nan"), float("inf"), -float("inf")):
        wrong = w.clone()
        wrong[h - 3] = value
        q, s = (t.float() for t in ops.rms_norm_quant(x, wrong, mode)[:2])
        assert torch.equal(q[:, : n * 128], want_q[:, : n * 128]) and torch.equal(s[:, :n], want_s[:, :n])
        if value != value:
            assert s[:, n].isnan().all() and q[:, n * 128:].isnan().all()
        else:
            assert (s[:, n] == float("inf")).all() and q[:, at].isnan().all() and not q[:, n * 128:][:, ~at[n * 128:]].any()
    # before the norm: 1 / rms is NaN, or it is zero and an infinity times that is NaN
    bad = x.clone()
    bad[1, 5], bad[3, h - 1] = float("nan"), float("inf")
    q, s = (t.float() for t in ops.rms_norm_quant(bad, w, mode)[:2])
    assert s[1].isnan().all() and q[1].isnan().all() and s[3, n].isnan() and q[3, n * 128:].isnan().all()
    assert s[3, :n].isfinite().all() and not q[3, : n * 128].any()
    assert torch.equal(q[[0, 2, 4]], want_q[[0, 2, 4]]) and torch.equal(s[[0, 2, 4]], want_s[[0, 2, 4]])


@pytest.mark.parametrize("device", DEVICES)
def test_norm_shapes(device):
    """Leading dimensions, no rows, rows that start anywhere in memory."""
    g = gen(device, 5)
    x, w = randn(g, 2, 3, 128, dtype=BF), randn(g, 128, dtype=BF)
    y, total = ops.add_rms_norm(x, x, w)
    flat = ops.add_rms_norm(x.view(6, 128), x.view(6, 128), w)
    assert y.shape == x.shape and torch.equal(y.view(6, 128), flat[0]) and torch.equal(total.view(6, 128), flat[1])
    q, s, _, _ = ops.rms_norm_quant(x, w, 3)
    assert q.shape == x.shape and s.shape == (2, 3, 1) and ops.rms_norm_quant(x, w, 2)[1].shape == (2, 3)
    assert ops.rms_norm(x[0, 0], w).shape == (128,)
    empty = x[:0]
    assert ops.rms_norm(empty, w).shape == (0, 3, 128) and ops.rms_norm_quant(empty, w, 4)[1].shape == (0, 3, 1)
    if cam_ops.native_loaded():
        leaf = w.clone().requires_grad_()
        (dw,) = torch.autograd.grad(ops.rms_norm(empty, leaf).float().sum(), leaf)
        assert not dw.any()
    for shift in (1, 3):  # in elements: not even 16-byte aligned
        buf = torch.zeros(6 * 128 + shift, dtype=BF, device=device)
        view = buf[shift:].view(6, 128)
        view.copy_(x.view(6, 128))
        # another order of the same sums: within twice the error of one
        a, b = ops.rms_norm(view, w).double(), ops.rms_norm(x.view(6, 128), w).double()
        assert ((a - b).abs() <= 2 * norm_tol(b, BF)).all()
        q, s, _, _ = ops.rms_norm_quant(view, w, 2)
        top = b.abs().amax(-1)
        within(s, top / 127, top / 127 * (half_step(BF)[0] + 2.0 ** -16), "scales")  # b is rounded to 16 bits
        assert (q.abs().amax(-1) == 127).all()


# ------------------------------------------------------------------------------------------------
# Routing
# ------------------------------------------------------------------------------------------------
ROUTES = {
    "softmax": (16, dict(k=4)),
    "one expert": (1, dict(k=1)),
    "odd": (37, dict(k=5)),
    "softmax as it is": (60, dict(k=6, renormalize=False, scale=1.5)),
    "all of them": (8, dict(k=8)),
    "best group": (64, dict(k=3, num_groups=4, topk_groups=2)),
    "odd groups": (90, dict(k=6, num_groups=6, topk_groups=3)),
    "sigmoid": (128, dict(k=8, score="sigmoid")),
    "sigmoid as it is": (40, dict(k=4, score="sigmoid", renormalize=False)),
    "two best of a group": (256, dict(k=8, score="sigmoid", num_groups=8, topk_groups=4, group_top=2, scale=2.5)),
    "two best, softmax": (48, dict(k=4, num_groups=8, topk_groups=3, group_top=2)),
    "groups of one": (32, dict(k=4, num_groups=32, topk_groups=9, group_top=2)),
    "many": (1024, dict(k=32, score="sigmoid")),
    "many groups": (1000, dict(k=10, num_groups=20, topk_groups=7, group_top=2)),
    "twelve lanes": (384, dict(k=8, score="sigmoid", num_groups=6, topk_groups=2, group_top=1)),
}


def masked_logits(g, t, e, dtype):
    """Rows with equal logits, with masked experts, with few that are left, with none."""
    x = randn(g, t, e, dtype=dtype)
    x[1] = 0.5
    x[2, ::2] = float("-inf")
    x[3, 1:] = float("-inf")
    x[4] = float("-inf")
    x[5] = torch.finfo(dtype).min
    x[6, 0], x[6, -1] = -0.0, 0.0
    x[7] = x[7] * 40
    x[8] = -x[8].abs() * 60 - 20
    return x


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("name", list(ROUTES))
def test_route(device, dtype, with_bias, name):
    e, kw = ROUTES[name]
    g = gen(device, e)
    t = 24
    x = masked_logits(g, t, e, dtype)
    bias = None
    if with_bias:
        bias = 0.1 * randn(g, e)
        bias[e // 2] = float("-inf") if e > kw["k"] * 2 else 0.0
    idx, w = ops.moe_route(x, bias=bias, **kw)
    idx64, w64 = route64(x, bias=bias, **kw)
    assert idx.dtype == torch.int64 and w.dtype == torch.float32
    assert torch.equal(idx, idx64)
    # logits of up to 240 apart: their exponents are rounded by that many u more
    within(w, w64, route_weight_tol(w64) * 4, "weights")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score,group_top", [("sigmoid", 2), ("softmax", 1), ("softmax", 2)])
@pytest.mark.parametrize("e,groups,open_groups,k", [(34, 2, 1, 5), (126, 2, 1, 9), (252, 4, 3, 8), (300, 4, 2, 7), (320, 4, 1, 3), (510, 5, 2, 6), (999, 3, 2, 12), (21, 7, 4, 2)])
def test_route_groups_that_end_inside_a_lane(device, dtype, score, group_top, e, groups, open_groups, k):
    g = gen(device, e + k)
    x, bias = masked_logits(g, 13, e, dtype), 0.1 * randn(g, e)
    kw = dict(k=k, score=score, num_groups=groups, topk_groups=open_groups, group_top=group_top)
    for b in (None, bias):
        idx, w = ops.moe_route(x, bias=b, **kw)
        idx64, w64 = route64(x, bias=b, **kw)
        assert torch.equal(idx, idx64)
        within(w, w64, route_weight_tol(w64) * 4, "weights")


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(ROUTES))
def test_route_gradient(device, dtype, name):
    e, kw = ROUTES[name]
    g = gen(device, e + 1)
    t = 21
    x = randn(g, t, e, dtype=dtype, scale=2.0)
    if kw["k"] < e:
        x[2, 1:] = float("-inf")
    x[3] = float("-inf")
    x.requires_grad_()
    idx, w = ops.moe_route(x, **kw)
    assert not idx.requires_grad
    dw = randn(g, *w.shape)
    (dx,) = torch.autograd.grad(w, x, dw)
    part = {n: kw[n] for n in ("score", "renormalize", "scale") if n in kw}
    live = torch.arange(t, device=device) != 3
    d, size = route_grad64(dw[live], x.detach()[live], idx[live], **part)
    half, tiny = half_step(dtype)
    within(dx[live], d, d.abs() * half + size * 256 * U + tiny, "dlogits")
    assert not dx[3].any()


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient_against_differences(device, score, renormalize):
    g = gen(device, 6)
    x = (randn(g, 4, 12) + 3 * torch.arange(12, device=device).remainder(5)).requires_grad_()  # choices that small steps do not change
    idx, w = ops.moe_route(x, 3, None, score, renormalize=renormalize, scale=2.0)
    dw = randn(g, 4, 3)
    (dx,) = torch.autograd.grad(w, x, dw)
    v, a = randn(g, 4, 12), 2.0 ** -6
    with torch.no_grad():
        hi, lo = (ops.moe_route(x + sign * a * v, 3, None, score, renormalize=renormalize, scale=2.0) for sign in (1, -1))
    if not (torch.equal(hi[0], idx) and torch.equal(lo[0], idx)):
        order = [r for r in range(4) if torch.equal(hi[0][r], idx[r]) and torch.equal(lo[0][r], idx[r])]
    else:
        order = list(range(4))
    assert len(order) >= 2
    want = float((dx.double() * v.double())[order].sum())
    got = float((((hi[1] - lo[1]).double() / (2 * a)) * dw.double())[order].sum())
    # a^2 v^3 of third derivatives below 1, twelve roundings of weights up to 2 over 2 a
    assert abs(got - want) <= 2.0 ** -8 * (1 + abs(want))


@pytest.mark.parametrize("device", DEVICES)
def test_route_special_rows(device):
    g = gen(device, 7)
    x = randn(g, 5, 16)
    x[0, 3] = float("nan")
    x[1, 4] = float("inf")
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(16, device=device)):
            idx, w = ops.moe_route(x, 4, bias, score)
            assert w[0].isnan().all() and ((idx >= -1) & (idx < 16)).all() and not (idx[0] == 3).any()
            assert w[2:].isfinite().all() and torch.equal(idx[2:], ops.moe_route(x[2:], 4, bias, score)[0])
    idx, w = ops.moe_route(x, 4, None, "sigmoid")
    assert idx[1, 0] == 4 and w[1].isfinite().all()
    assert ops.moe_route(x[:0], 4)[0].shape == (0, 4)
    # scores that fp32 cannot tell apart, or cannot hold, keep their order and their ratios
    far = torch.tensor([[-200.0, -201.0, -199.0, -250.0], [60.0, 59.0, 61.0, 20.0]], device=device)
    idx, w = ops.moe_route(far, 2, None, "sigmoid")
    assert idx.tolist() == [[2, 0], [2, 0]]
    within(w[0], torch.softmax(far[0, [2, 0]].double(), -1), torch.full_like(w[0], 2.0 ** -18).double())
    # with a bias ranks are scores: those near 1 are told apart in 64 bits, and equal ones go to the lowest index
    near = torch.tensor([[18.0, 19.0, 20.0, 17.0, 45.0, 44.0]], device=device)
    assert ops.moe_route(near, 6, torch.zeros(6, device=device), "sigmoid")[0].tolist() == [[4, 5, 2, 1, 0, 3]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("e", [16, 60])
def test_route_groups_of_rows_that_are_not_finite(device, dtype, score, with_bias, group_top, e):
    """A softmax of NaN or infinity has no value: where groups or experts are ranked by it nothing is chosen; elsewhere logits rank as they
    are and NaN is left out."""
    g = gen(device, 13)
    x, bias = randn(g, 7, e, dtype=dtype), 0.1 * randn(g, e) if with_bias else None
    x[0, 3], x[1, 4], x[2] = float("nan"), float("inf"), float("nan")
    x[3, 1] = x[3, e - 2] = float("inf")
    x[4, : e // 4] = -float("inf")
    kw = dict(bias=bias, score=score, num_groups=4, topk_groups=2, group_top=group_top)
    idx, w = ops.moe_route(x, 3, **kw)
    want, w64 = route64(x, 3, **kw)
    if score == "softmax" and (with_bias or group_top == 2):
        want[:4] = -1
    assert torch.equal(idx, want)
    assert w[[0, 1, 2, 3] if score == "softmax" else [0, 2]].isnan().all()
    within(w[4:], w64[4:], route_weight_tol(w64[4:]), "weights")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_close_scores(device, dtype):
    """Many rows with sigmoid and bias: neighbours closer than fp32 can tell are ranked in 64 bits."""
    g = gen(device, 8)
    x = randn(g, 3000, 256, dtype=dtype)
    bias = 0.05 * randn(g, 256)
    idx, _ = ops.moe_route(x, 8, bias, "sigmoid", 8, 4, 2)
    rank = torch.sigmoid(x.double()) + bias.double()
    two = rank.view(-1, 8, 32).topk(2, -1).values.sum(-1)
    keep = two.sort(dim=-1, descending=True, stable=True).indices[:, :4]
    mask = torch.zeros_like(two, dtype=torch.bool).scatter_(1, keep, True).repeat_interleave(32, 1)
    want = rank.masked_fill(~mask, -9.0).sort(dim=-1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(idx, want)


# ------------------------------------------------------------------------------------------------
# Rows grouped by expert and brought back
# ------------------------------------------------------------------------------------------------
def routing(g, t, k, e, drop=0.0, same=False):
    idx = torch.stack([torch.randperm(max(e, k), generator=g, device=g.device)[:k] for _ in range(t)]) if t else torch.zeros(0, k, dtype=torch.long, device=g.device)
    idx = torch.where(idx < e, idx, torch.full_like(idx, -1))
    if same:
        idx[:, 1:] = idx[:, :1]
    if drop:
        idx = torch.where(torch.rand(t, k, generator=g, device=g.device) < drop, torch.full_like(idx, -1), idx)
    return idx


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [*DTYPES, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("t,k,e,h", [(1, 1, 1, 8), (1, 8, 256, 128), (5, 2, 3, 7), (33, 4, 8, 40), (130, 3, 1024, 1000), (64, 32, 40, 24), (700, 6, 17, 264)])
def test_group_rows(device, dtype, t, k, e, h):
    g = gen(device, t + h)
    x = randn(g, t, h, scale=20.0)
    x = x.round().clamp(-127, 127).to(dtype) if dtype == torch.int8 else x.to(dtype)
    for drop, ints in ((0.0, torch.int64), (0.4, torch.int32), (1.0, torch.int64)):
        idx = routing(g, t, k, e, drop).to(ints)
        for scales in (None, torch.rand(t, generator=g, device=device), torch.rand(t, 5, generator=g, device=device)):
            rows, rs, off, slots = ops.moe_group_rows(x, idx, e, scales)
            rows64, rs64, off64, slots64 = group64(x, idx, e, scales)
            assert rows.dtype == dtype and off.dtype == slots.dtype == torch.int32
            assert torch.equal(off, off64) and torch.equal(slots, slots64) and torch.equal(rows.float(), rows64)
            assert rs.numel() == 0 if scales is None else torch.equal(rs, rs64)


@pytest.mark.parametrize("device", DEVICES)
def test_group_rows_odd_ids(device):
    """Ids of other ranks, of no expert, past 32 bits; one expert twice for a token; no tokens."""
    g = gen(device, 9)
    x = randn(g, 4, 16, dtype=BF)
    idx = torch.tensor([[0, 7], [2 ** 32, -1], [3, 3], [-2 ** 40, 2]], device=device)
    rows, _, off, slots = ops.moe_group_rows(x, idx, 4)
    assert off.tolist() == [0, 1, 1, 2, 4] and slots.tolist() == [[0, -1], [-1, -1], [2, 3], [-1, 1]]
    assert torch.equal(rows[:4], x[[0, 3, 2, 2]]) and not rows[4:].any()
    rows, rs, off, slots = ops.moe_group_rows(x[:0], idx[:0], 4, torch.zeros(0, 2, device=device))
    assert rows.shape == (0, 16) and rs.shape == (0, 2) and off.tolist() == [0] * 5 and slots.shape == (0, 2)
    assert ops.moe_ungroup_rows(rows, slots).shape == (0, 16)


UNGROUPS = [(1, 1, 8), (3, 2, 7), (17, 9, 40), (40, 3, 1000), (9, 8, 1032), (5, 32, 2050), (260, 2, 264), (12, 4, 4096)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k,h", UNGROUPS)
@pytest.mark.parametrize("weighted,with_residual", [(True, False), (True, True), (False, False), (False, True)])
def test_ungroup_rows_and_gradients(device, dtype, t, k, h, weighted, with_residual):
    g = gen(device, t * k + h)
    m = t * k + 5  # rows that nobody brings back: the rest of a receive buffer
    slots = torch.randperm(m, generator=g, device=device)[: t * k].to(torch.int32).view(t, k)
    slots = torch.where(torch.rand(t, k, generator=g, device=device) < 0.2, torch.full_like(slots, -1), slots)
    rows = randn(g, m, h, dtype=dtype)
    w = torch.rand(t, k, generator=g, device=device) if weighted else None
    res = randn(g, t, h, dtype=dtype) if with_residual else None
    valid = slots >= 0
    picked = torch.where(valid[..., None], rows.double()[slots.clamp(min=0).long()], 0.0)
    w64 = torch.where(valid, w.double() if weighted else 1.0, 0.0)
    terms = picked * w64[..., None]
    want = terms.sum(1) + (res.double() if with_residual else 0.0)
    size = terms.abs().sum(1) + (res.double().abs() if with_residual else 0.0)
    half, tiny = half_step(dtype)
    with torch.no_grad():
        out = ops.moe_ungroup_rows(rows, slots, w, res)
    within(out, want, want.abs() * half + size * (k + 3) * U + tiny, "out")
    if not cam_ops.native_loaded():
        return
    leaves = [None if v is None else v.clone().requires_grad_() for v in (rows, w, res)]
    again = ops.moe_ungroup_rows(leaves[0], slots, leaves[1], leaves[2])
    assert torch.equal(again, out)
    dout = randn(g, t, h, dtype=dtype)
    given = [v for v in leaves if v is not None]
    grads = list(torch.autograd.grad(again, given, dout))
    d64 = torch.zeros(m, h, dtype=torch.float64, device=device)
    d64[slots[valid].long()] = (dout.double()[:, None] * w64[..., None])[valid]
    within(grads[0], d64, d64.abs() * (half + 2 * U) + tiny, "drows")
    if weighted:
        terms = picked * dout.double()[:, None]
        # a thread adds at most a 32nd of a row (a warp's share of up to 1024 values, a block's of more), then the threads
        within(grads[1], terms.sum(-1), terms.abs().sum(-1) * (h / 16 + 64) * U + 2.0 ** -140, "dweights")
        only = leaves[1].detach().clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(ops.moe_ungroup_rows(rows, slots, only, res), only, dout)[0], grads[1])
    if with_residual:
        assert torch.equal(grads[-1], dout)


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [7, 40, 1032])
@pytest.mark.parametrize("weighted", [False, True])
def test_rows_that_no_gradient_reads_are_not_kept(device, dtype, h, weighted):
    """Weights without a gradient, or none: the rows may change and their memory may go before the backward pass."""
    g = gen(device, h)
    z = randn(g, 6, h, dtype=dtype).requires_grad_()
    slots = torch.tensor([[0, 4], [-1, 2], [5, 1]], device=device, dtype=torch.int32)
    w = torch.rand(3, 2, generator=g, device=device) if weighted else None
    dout = randn(g, 3, h, dtype=dtype)
    rows = z * 1
    held = weakref.ref(rows.untyped_storage())
    out = ops.moe_ungroup_rows(rows, slots, w)
    with torch.no_grad():
        rows.add_(1)
    del rows
    gc.collect()
    assert held() is None
    (got,) = torch.autograd.grad(out, z, dout)
    weights = torch.ones(3, 2, device=device) if w is None else w
    want, _ = ops.moe_ungroup_rows_backward(dout, z.detach(), slots, weights)
    assert torch.equal(got, want)
    # the operator itself: rows [M, 0] stand for their number, but not where they are read
    none = z.detach()[:, :0].contiguous()
    assert torch.equal(ops.moe_ungroup_rows_backward(dout, none, slots, weights, True, False)[0], want)
    with pytest.raises(RuntimeError, match="rows must be"):
        ops.moe_ungroup_rows_backward(dout, none, slots, weights)
    with pytest.raises(RuntimeError, match="rows must be"):
        ops.moe_ungroup_rows_backward(dout[:, :0].contiguous(), none, slots, weights, True, False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [7, 8, 264, 2048, 2050])
def test_ungroup_weight_gradients_of_places_without_a_row(device, dtype, h):
    """They are zero whatever the token's gradient holds."""
    g = gen(device, h)
    rows, w = randn(g, 6, h, dtype=dtype), torch.rand(2, 3, generator=g, device=device)
    slots = torch.tensor([[0, -1, 9], [-1, -1, 3]], device=device, dtype=torch.int32)
    dout = torch.ones(2, h, device=device, dtype=dtype)
    dout[0, h // 2], dout[1, h - 1] = float("inf"), float("nan")
    _, dw = ops.moe_ungroup_rows_backward(dout, rows, slots, w)
    none = (slots < 0) | (slots >= 6)
    assert not dw[none].any() and not dw[~none].isfinite().any()


@native
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k,e,h", [(1, 1, 1, 8), (6, 3, 4, 7), (130, 8, 16, 264)])
def test_group_rows_gradient(device, dtype, t, k, e, h):
    g = gen(device, 11)
    idx = routing(g, t, k, e, 0.2)
    x = randn(g, t, h, dtype=dtype).requires_grad_()
    rows, _, off, slots = ops.moe_group_rows(x, idx, e)
    assert not off.requires_grad and not slots.requires_grad
    drows = randn(g, t * k, h, dtype=dtype)
    (dx,) = torch.autograd.grad(rows, x, drows)
    terms = torch.where((slots >= 0)[..., None], drows.double()[slots.clamp(min=0).long()], 0.0)
    half, tiny = half_step(dtype)
    within(dx, terms.sum(1), terms.sum(1).abs() * half + terms.abs().sum(1) * (k + 1) * U + tiny, "dx")


@native
@pytest.mark.parametrize("device", DEVICES)
def test_one_expert_twice_for_a_token(device):
    """The gradients of both places meet."""
    g = gen(device, 12)
    idx = routing(g, 9, 3, 4, same=True)
    x, w = randn(g, 9, 24).requires_grad_(), torch.rand(9, 3, generator=g, device=device).requires_grad_()
    rows, _, _, slots = ops.moe_group_rows(x, idx, 4)
    out = ops.moe_ungroup_rows(rows * 2, slots, w)
    dout = randn(g, 9, 24)
    dx, dw = torch.autograd.grad(out, (x, w), dout)
    total = w.detach().double().sum(-1, keepdim=True)
    within(out, 2 * x.detach().double() * total, (2 * x.detach().double() * total).abs() * 8 * U + 1e-30)
    within(dx, 2 * dout.double() * total, (2 * dout.double() * total).abs() * 8 * U + 1e-30)
    dots = (2 * x.detach().double() * dout.double())
    within(dw, dots.sum(-1, keepdim=True).expand(9, 3), (dots.abs().sum(-1, keepdim=True) * 66 * U).expand(9, 3))


# ------------------------------------------------------------------------------------------------
# Refusals
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    i64 = torch.int64

    def refused(match, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*args, **kw)
    refused("weight must be", ops.rms_norm, z(4, 16), z(15))
    refused("weight must be", ops.rms_norm, z(4, 16), z(16, dtype=HF))
    refused("at most 16384", ops.rms_norm, z(1, 16392), z(16392))
    refused("bfloat16, float16 or float32", ops.rms_norm, z(4, 16, dtype=torch.float64), z(16, dtype=torch.float64))
    refused("contiguous", ops.rms_norm, z(16, 4).t(), z(16))
    refused("eps", ops.rms_norm, z(4, 16), z(16), -1.0)
    refused(r"must be \[\.\.\., h\]", ops.rms_norm, z(4, 0), z(0))
    refused("residual must be", ops.add_rms_norm, z(4, 16), z(3, 16), z(16))
    refused("residual must be", ops.add_rms_norm, z(4, 16), z(4, 16, dtype=HF), z(16))
    refused("quant_mode must be", ops.rms_norm_quant, z(4, 128), z(128), 0)
    refused("multiple of 128", ops.rms_norm_quant, z(4, 136), z(136), 3)
    refused("rstd", ops.rms_norm_backward, z(4, 16), None, z(4, 16), z(16), z(3, dtype=FL))
    refused("dsum", ops.rms_norm_backward, z(4, 16), z(4, 8), z(4, 16), z(16), z(4, dtype=FL))
    refused(r"k 0 outside", ops.moe_route, z(4, 8), 0)
    refused(r"k 9 outside", ops.moe_route, z(4, 8), 9)
    refused("at most 1024", ops.moe_route, z(4, 1025), 2)
    refused("k 33 outside", ops.moe_route, z(4, 64), 33)
    refused("logits must be", ops.moe_route, z(8), 1)
    refused("score must be", ops.moe_route, z(4, 8), 2, None, "tanh")
    refused("bias must be", ops.moe_route, z(4, 8), 2, z(8))
    refused("bias must be", ops.moe_route, z(4, 8), 2, z(7, dtype=FL))
    refused("groups of equal size", ops.moe_route, z(4, 8), 2, None, "softmax", 3, 1)
    refused("groups of equal size", ops.moe_route, z(4, 66), 2, None, "softmax", 33, 3)
    refused("topk_groups", ops.moe_route, z(4, 8), 2, None, "softmax", 4, 5)
    refused("k 3 of the 2 experts", ops.moe_route, z(4, 8), 3, None, "softmax", 4, 1)
    refused("group_top", ops.moe_route, z(4, 8), 2, None, "softmax", 2, 1, 3)
    refused("dweights must be", ops.moe_route_backward, z(4, 3, dtype=FL), z(4, 8), z(4, 2, dtype=i64))
    refused("topk_idx must be", ops.moe_route_backward, z(4, 2, dtype=FL), z(4, 8), z(4, 2, dtype=torch.int32))
    refused(r"x must be \[T, h\]", ops.moe_group_rows, z(4, 8), z(5, 2, dtype=i64), 4)
    refused("int64 or int32", ops.moe_group_rows, z(4, 8), z(4, 2), 4)
    refused("choices per token", ops.moe_group_rows, z(4, 8), z(4, 33, dtype=i64), 4)
    refused("choices per token", ops.moe_group_rows, z(4, 8), z(4, 0, dtype=i64), 4)
    refused("1 to 1024", ops.moe_group_rows, z(4, 8), z(4, 2, dtype=i64), 1025)
    refused("1 to 1024", ops.moe_group_rows, z(4, 8), z(4, 2, dtype=i64), 0)
    refused("must be bfloat16", ops.moe_group_rows, z(4, 8, dtype=torch.float64), z(4, 2, dtype=i64), 4)
    refused("scales must be", ops.moe_group_rows, z(4, 8), z(4, 2, dtype=i64), 4, z(3, dtype=FL))
    refused("scales must be", ops.moe_group_rows, z(4, 8), z(4, 2, dtype=i64), 4, z(4, 0, dtype=FL))
    refused("contiguous", ops.moe_group_rows, z(8, 4).t(), z(4, 2, dtype=i64), 4)
    refused("slots must be", ops.moe_ungroup_rows, z(8, 16), z(4, 2, dtype=i64))
    refused("topk_weights must be", ops.moe_ungroup_rows, z(8, 16), z(4, 2, dtype=torch.int32), z(4, 2))
    refused("residual must be", ops.moe_ungroup_rows, z(8, 16), z(4, 2, dtype=torch.int32), None, z(4, 15))
    refused("rows must be", ops.moe_ungroup_rows, z(8), z(4, 2, dtype=torch.int32))
    refused("dout must be", ops.moe_ungroup_rows_backward, z(3, 16), z(8, 16), z(4, 2, dtype=torch.int32))
    # nothing above left anything behind
    assert ops.rms_norm(z(4, 16), z(16)).shape == (4, 16)


@native
@pytest.mark.parametrize("device", DEVICES)
def test_what_has_no_gradient(device):
    x = torch.ones(4, 128, dtype=BF, device=device, requires_grad=True)
    w = torch.ones(128, dtype=BF, device=device)
    idx = torch.zeros(4, 1, dtype=torch.int64, device=device)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(ops.rms_norm_quant(x, w, 3, None, 1e-6, True)[3].sum(), x)
    scales = torch.ones(4, 1, device=device, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.moe_group_rows(x.detach(), idx, 2, scales)
    y = ops.rms_norm(x, w)
    (g,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), x)
    with torch.no_grad():
        assert not ops.rms_norm(x, w).requires_grad
