"""Norm, routing and rows grouped by expert on the GPU: sizes past 32 bits, graphs, streams, threads, memory of a dispatch."""
import threading

import pytest
import torch

from layer_cases import group64, norm64, norm_grad_tol, norm_grads64, norm_tol, weight_grad_tol, within
from umdk_original_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def make(t=50, h=264, e=8, k=3, dtype=BF, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, d=dtype: torch.randn(*s, device=DEV, generator=g).to(d)  # noqa: E731
    return dict(x=r(t, h), residual=r(t, h), weight=r(h), gate=r(e, h) * h ** -0.5, bias=0.1 * r(e, d=torch.float32), dout=r(t, h), ds=r(t, h),
                e=e, k=k)


def chain(c, x, residual, weight, gate):
    """One pass through all of them, as a block uses them (the experts double their rows)."""
    y, s = ops.add_rms_norm(x, residual, weight)
    idx, w = ops.moe_route(y @ gate.t(), c["k"], c["bias"], "sigmoid", 4, 2, 2)
    rows, _, off, slots = ops.moe_group_rows(y, idx, c["e"])
    out = ops.moe_ungroup_rows(rows * 2, slots, w, s)
    return out, s, idx, w, rows, off, slots


def step(c, leaves):
    res = chain(c, *leaves)
    return [t.detach() for t in res] + list(torch.autograd.grad(res[:2], leaves, (c["dout"], c["ds"])))


def leaves_of(c):
    return [c[n].clone().requires_grad_() for n in ("x", "residual", "weight", "gate")]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


def test_capture_and_replay():
    """Forward and backward in one CUDA graph, replayed with other data; two graphs that are replayed in turn; a side stream."""
    c = make()
    leaves = leaves_of(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(c, leaves)
    torch.cuda.current_stream().wait_stream(side)
    want = step(c, leaves)
    assert same(first, want)
    del first
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    others = [leaves, leaves_of(make(seed=4))]
    for g, l in zip(graphs, others):
        with torch.cuda.graph(g):
            outs.append(step(c, l))
    c2 = make(seed=9)
    with torch.no_grad():
        for a, n in zip(leaves, ("x", "residual", "weight", "gate")):
            a.copy_(c2[n])
    for n in ("bias", "dout", "ds"):
        c[n].copy_(c2[n])
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i].replay()
        for i in (0, 1):
            assert same([t.clone() for t in outs[i]], step(c, others[i]))


def test_capture_beside_an_eager_graph_is_refused():
    c = make()
    cases = {
        "rms_norm": lambda t: ops.rms_norm(t, c["weight"]),
        "add_rms_norm": lambda t: ops.add_rms_norm(c["x"], t, c["weight"])[1],
        "moe_route": lambda t: ops.moe_route(t, 2)[1],
        "moe_group_rows": lambda t: ops.moe_group_rows(t, torch.zeros(50, 1, dtype=torch.int64, device=DEV), 2)[0],
        "moe_ungroup_rows": lambda t: ops.moe_ungroup_rows(t, torch.arange(50, device=DEV, dtype=torch.int32)[:, None].contiguous()),
    }
    for name, fn in cases.items():
        fn(c["x"])  # whatever has to be loaded is
        leaf = c["x"].clone().requires_grad_()
        eager = fn(leaf)  # holds the leaf's accumulation node
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=f"{name} is captured.*let go of its outputs"):
            with torch.cuda.graph(g):
                fn(leaf)
        del eager
        g = torch.cuda.CUDAGraph()
        idx = torch.zeros(50, 1, dtype=torch.int64, device=DEV)
        slots = torch.arange(50, device=DEV, dtype=torch.int32)[:, None].contiguous()
        fn = {"moe_group_rows": lambda t: ops.moe_group_rows(t, idx, 2)[0], "moe_ungroup_rows": lambda t: ops.moe_ungroup_rows(t, slots)}.get(name, fn)
        ones = torch.ones_like(fn(c["x"]))
        with torch.cuda.graph(g):
            out = fn(leaf)
            grad, = torch.autograd.grad(out, leaf, ones)
        g.replay()
        again = fn(leaf)
        assert torch.equal(out, again) and torch.equal(grad, torch.autograd.grad(again, leaf, ones)[0])


def test_waits_for_another_stream():
    """The kernels may start before the one ahead of them on their stream has finished, but not before an event they wait for."""
    c = make()
    leaves = leaves_of(c)
    want = step(c, leaves)
    late = [torch.zeros_like(t).requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(c, leaves)  # kernels ahead on this stream
    with torch.cuda.stream(side), torch.no_grad():
        torch.cuda._sleep(2_000_000)  # about a millisecond
        for a, b in zip(late, leaves):
            a.copy_(b)
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want) and same(step(c, late), want)


def test_calls_from_two_host_threads():
    c = make(seed=3)
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            leaves = leaves_of(c)
            for _ in range(20):
                got[i] = step(c, leaves)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    want = step(c, leaves_of(c))
    assert same(got[0], want) and same(got[1], want)


def test_norm_past_32_bits():
    """2^31 values and more: the last rows are what they are on their own."""
    h, rows = 8192, 2 ** 18 + 700
    x = torch.randn(4096, h, device=DEV).to(BF).repeat(65, 1)[:rows]
    w = torch.randn(h, device=DEV).to(BF).requires_grad_()
    x.requires_grad_()
    y = ops.rms_norm(x, w)
    part = x.detach()[-300:].clone().requires_grad_()
    y2 = ops.rms_norm(part, w)
    assert torch.equal(y[-300:], y2)
    dy = torch.randn(300, h, device=DEV).to(BF)
    full = torch.zeros_like(y)
    full[-300:] = dy
    dx, dw = torch.autograd.grad(y, (x, w), full)
    dx2, dw2 = torch.autograd.grad(y2, (part, w), dy)
    assert torch.equal(dx[-300:], dx2) and not dx[:1000].any()
    # the same rows in other blocks: half a step of bf16 each, and the order of 300 sums in fp32
    assert ((dw - dw2).abs().double() <= dw2.abs().double() * 2.0 ** -7 + 300 * 2.0 ** -20).all()
    del y, y2, full, dx
    q, s, _, _ = ops.rms_norm_quant(x.detach(), w.detach(), 3)
    q2, s2, _, _ = ops.rms_norm_quant(part.detach(), w.detach(), 3)
    assert torch.equal(q[-300:].view(torch.int8), q2.view(torch.int8)) and torch.equal(s[-300:], s2)


@pytest.mark.parametrize("dtype,residual,weight", [(BF, BF, BF), (torch.float16, torch.float32, torch.float16), (torch.float32, torch.float32, torch.float32),
                                                   (BF, None, torch.float32)])
@pytest.mark.parametrize("rows,h", [(40001, 72), (20003, 504), (11000, 520), (9999, 1000), (6007, 2056), (3001, 4096), (1301, 7168), (701, 8200), (700, 16384), (5003, 333)])
def test_norm_gradients_of_many_rows(dtype, residual, weight, rows, h):
    """More than two turns of all blocks: rows are loaded ahead (or, with an odd width, not), in both directions and with both gradients."""
    g = torch.Generator(device=DEV).manual_seed(h)
    r = lambda *s, d: torch.randn(*s, device=DEV, generator=g).to(d)  # noqa: E731
    x, w, dy = r(rows, h, d=dtype), r(h, d=weight), r(rows, h, d=dtype)
    res, ds = (None, None) if residual is None else (r(rows, h, d=residual), r(rows, h, d=residual))
    leaves = [t.requires_grad_() for t in (x, res, w) if t is not None]
    out = (ops.rms_norm(x, w),) if res is None else ops.add_rms_norm(x, res, w)
    grads = torch.autograd.grad(out, leaves, [t for t in (dy, ds) if t is not None])
    with torch.no_grad():
        y64, total, _ = norm64(x, res, w, 1e-6)
        within(out[0].detach(), y64, norm_tol(y64, dtype), "y")
        del y64
        assert res is None or torch.equal(out[1], total)
        d, size, dw, dw_size = norm_grads64(dy, ds, total, w, 1e-6)
        within(grads[0], d, norm_grad_tol(d, size, dtype), "dx")
        if res is not None:
            within(grads[1], d, norm_grad_tol(d, size, residual), "dresidual")
        within(grads[-1], dw, weight_grad_tol(dw, dw_size, rows, weight), "dweight")
        # a row's numbers do not depend on how many there are
        few = ops.rms_norm_train(x[5:9].contiguous(), None if res is None else res[5:9].contiguous(), w)
        if h % 8 == 0:
            assert torch.equal(few[0], out[0][5:9])
            back = ops.rms_norm_backward(dy[5:9].contiguous(), None if ds is None else ds[5:9].contiguous(), total[5:9].contiguous(), w, few[2])
            assert torch.equal(back[0], grads[0][5:9])


@pytest.mark.parametrize("dtype,residual", [(BF, BF), (torch.float16, torch.float32), (torch.float32, None)])
@pytest.mark.parametrize("rows,h,shift", [(2003, 255, 0), (2003, 257, 0), (2001, 256, 1), (301, 4097, 0), (201, 8191, 0), (201, 8193, 0), (201, 8192, 1), (101, 12008, 3)])
def test_norm_value_by_value(dtype, residual, rows, h, shift):
    g = torch.Generator(device=DEV).manual_seed(h + shift)
    r = lambda n, d: torch.randn(n + shift, device=DEV, generator=g).to(d)[shift:]  # noqa: E731
    x, w = r(rows * h, dtype).view(rows, h), r(h, dtype)
    res = None if residual is None else r(rows * h, residual).view(rows, h)
    y64, total, _ = norm64(x, res, w, 1e-6)
    y = ops.rms_norm(x, w) if res is None else ops.add_rms_norm(x, res, w)[0]
    within(y, y64, norm_tol(y64, dtype), "rows")
    q, s, kept, rows8 = ops.rms_norm_quant(x, w, 2, res, 1e-6, True)
    assert torch.equal(rows8, y) and (res is None or torch.equal(kept, total))
    rel = 40 * 2.0 ** -24  # of a value of y (32 u), a scale's division and product
    top = y64.abs().amax(-1)
    within(s, top / 127, top / 127 * rel, "scales")
    within(q.double() * s.double()[:, None], y64, s.double()[:, None] * (0.5 + 127 * 3 * rel), "values")


@pytest.mark.parametrize("h", [96, 203, 1024, 4096, 7168, 9001])
def test_norm_int8_rows_that_are_not_finite(h):
    """NaN, or an infinity before the norm: the scale is NaN; an infinity behind it: infinite.  The values are zero, other rows as without."""
    g = torch.Generator(device=DEV).manual_seed(h)
    x, w = torch.randn(9, h, device=DEV, generator=g), torch.rand(h, device=DEV, generator=g) + 0.5
    want = ops.rms_norm_quant(x, w, 2)
    bad = x.clone()
    bad[1, h - 1], bad[3, 0], bad[6] = float("nan"), float("inf"), float("-inf")
    q, s, _, _ = ops.rms_norm_quant(bad, w, 2)
    assert s[[1, 3, 6]].isnan().all() and not q[[1, 3, 6]].any()
    keep = [0, 2, 4, 5, 7, 8]
    assert torch.equal(q[keep], want[0][keep]) and torch.equal(s[keep], want[1][keep])
    for value in (float("nan"), float("inf")):
        wrong = w.clone()
        wrong[h // 2] = value
        q, s, _, y = ops.rms_norm_quant(x, wrong, 2, None, 1e-6, True)
        assert (s.isnan() if value != value else s.isinf()).all() and not q.any()
        assert y.isfinite().sum() == 9 * (h - 1)


@pytest.mark.parametrize("dtype,sums", [(BF, BF), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,h,shift", [(9001, 255, 0), (9001, 257, 0), (1201, 4097, 0), (601, 8191, 0), (601, 8193, 0), (4001, 256, 1), (4001, 264, 1),
                                          (601, 8192, 1), (601, 8200, 1)])
def test_norm_gradients_value_by_value(dtype, sums, rows, h, shift):
    """Odd widths, and rows that start off every boundary, where the threads' share of a row changes."""
    g = torch.Generator(device=DEV).manual_seed(h)
    r = lambda *s, d: torch.randn(*s, device=DEV, generator=g).to(d)  # noqa: E731
    total, dy, ds = (r(rows * h + shift, d=d)[shift:].view(rows, h) for d in (sums, dtype, sums))
    w = r(h, d=dtype)
    rstd = (total.double().square().mean(1) + 1e-6).rsqrt().float()
    dx, dres, dw = ops.rms_norm_backward(dy, ds, total, w, rstd, True, True, True)
    d, size, want, dw_size = norm_grads64(dy, ds, total, w, 1e-6)
    within(dx, d, norm_grad_tol(d, size, dtype), "dx")
    within(dx if sums == dtype else dres, d, norm_grad_tol(d, size, sums), "dresidual")  # one tensor where they are of one type
    within(dw, want, weight_grad_tol(want, dw_size, rows, dtype), "dweight")


@pytest.mark.parametrize("mode", [2, 3, 4])
def test_norm_quant_at_16_bytes(mode):
    """Operands at 16 bytes that are not at 32: the same bits."""
    def at_16(t):
        buf = torch.zeros(t.numel() + 8, device=DEV, dtype=t.dtype)
        return buf[8:].view(t.shape).copy_(t)
    x, r, w = (torch.randn(*s, device=DEV).to(BF) for s in ((300, 1280), (300, 1280), (1280,)))
    a, b = ops.rms_norm_quant(x, w, mode, r, 1e-6, True), ops.rms_norm_quant(at_16(x), at_16(w), mode, at_16(r), 1e-6, True)
    assert all(torch.equal(u.view(torch.int8) if u.dtype == torch.float8_e4m3fn else u, v.view(torch.int8) if v.dtype == torch.float8_e4m3fn else v) for u, v in zip(a, b))


def test_softmax_weights_and_their_gradient_are_of_one_softmax():
    """Two experts, weights as they are: the gradient of the first weight by the second logit is minus the product of both weights, to the
    bit, and the weights are an fp32 softmax."""
    d = torch.linspace(0.0, 12.0, 1 << 14, device=DEV)
    x = torch.stack([torch.zeros_like(d), -d], 1).contiguous().requires_grad_()
    idx, w = ops.moe_route(x, 2, None, "softmax", renormalize=False)
    assert torch.equal(idx, torch.tensor([0, 1], device=DEV).expand_as(idx))
    (dx,) = torch.autograd.grad(w, x, torch.tensor([1.0, 0.0], device=DEV).expand_as(w).contiguous())
    w = w.detach()
    assert torch.equal(dx[:, 1], -(w[:, 0] * w[:, 1]))
    # u = 2^-24: expf 2 u, of which the first weight takes the second's share, a sum, a reciprocal, and one product for the second
    want = torch.softmax(x.detach().double(), -1)
    share, u = want[:, 1:], 2.0 ** -24
    within(w, want, want * (torch.cat([2 + 2 * share, 5 + 2 * share], 1) * u))


@pytest.mark.parametrize("t,k,h,dtype", [(3000, 8, 2047, BF), (3000, 4, 1023, torch.float32), (2500, 2, 4095, torch.float16), (3000, 3, 8, BF), (1100, 32, 512, torch.float32)])
def test_many_rows_there_and_back(t, k, h, dtype):
    """Sizes at which every form of the kernels goes round: the identity of both directions, gradients against index arithmetic."""
    g = torch.Generator(device=DEV).manual_seed(t + h)
    idx = torch.rand(t, 40, device=DEV, generator=g).topk(k, -1).indices
    idx = torch.where(torch.rand(t, k, device=DEV, generator=g) < 0.1, torch.full_like(idx, -1), idx)
    x = torch.randn(t, h, device=DEV, generator=g).to(dtype).requires_grad_()
    rows, _, off, slots = ops.moe_group_rows(x, idx, 40)
    n, valid = int(off[-1]), slots >= 0
    assert n == int(valid.sum()) and not rows[n:].any()
    back = rows[slots.clamp(min=0).long()]
    assert torch.equal(back[valid], x[:, None].expand(-1, k, -1)[valid])
    results, w = torch.randn(t * k, h, device=DEV, generator=g).to(dtype).requires_grad_(), torch.rand(t, k, device=DEV, generator=g).requires_grad_()
    out = ops.moe_ungroup_rows(results, slots, w)
    dout, drows = torch.randn(t, h, device=DEV, generator=g).to(dtype), torch.randn(t * k, h, device=DEV, generator=g).to(dtype)
    dx, dres, dw = torch.autograd.grad((rows, out), (x, results, w), (drows, dout))
    half, tiny, u = {BF: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}[dtype], 2.0 ** -24, 2.0 ** -24
    at = slots.clamp(min=0).long()
    for got, terms in ((out, torch.where(valid[..., None], results.detach().double()[at] * w.detach().double()[..., None], 0.0)),
                       (dx, torch.where(valid[..., None], drows.double()[at], 0.0))):
        want = terms.sum(1)
        within(got.detach(), want, want.abs() * half + terms.abs().sum(1) * (k + 3) * u + tiny)
    want = torch.zeros(t * k, h, device=DEV, dtype=torch.float64)
    want[slots[valid].long()] = (dout.double()[:, None] * w.detach().double()[..., None])[valid]
    within(dres, want, want.abs() * (half + 2 * u) + tiny)
    terms = torch.where(valid[..., None], results.detach().double()[at], 0.0) * dout.double()[:, None]
    within(dw, terms.sum(-1), terms.abs().sum(-1) * (h / 16 + 64) * u + 2.0 ** -140)


def many_slots(t, k, m, g, drop=0.1):
    """Slots of t tokens among m rows, some of none; in every 512 rows some that nobody names, and the last ones."""
    free = torch.arange(m, device=DEV)
    free = free[(free % 512 > 2) & (free < m - 40)]
    slots = free[torch.randperm(free.numel(), device=DEV, generator=g)[: t * k]].to(torch.int32).view(t, k)
    return torch.where(torch.rand(t, k, device=DEV, generator=g) < drop, torch.full_like(slots, -1), slots)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("t,k,h", [(40000, 8, 16), (131072, 8, 8), (70000, 2, 21), (20000, 8, 1032), (16400, 8, 40)])
def test_gradients_of_many_rows_of_which_some_have_no_token(dtype, t, k, h):
    """More rows and slots than the blocks that write zeros look at in one go; rows of no slot lie everywhere.  Any alignment of the slots."""
    g = torch.Generator(device=DEV).manual_seed(h)
    m = t * k + t * k // 64 + 77
    slots = many_slots(t, k, m, g)
    w, dout, rows = torch.rand(t, k, device=DEV, generator=g), torch.randn(t, h, device=DEV, generator=g).to(dtype), torch.randn(m, h, device=DEV, generator=g).to(dtype)
    drows, dw = ops.moe_ungroup_rows_backward(dout, rows, slots, w)
    valid = slots >= 0
    unused = torch.ones(m, dtype=torch.bool, device=DEV)
    unused[slots[valid].long()] = False
    assert unused[-40:].all() and unused.view(-1)[: m // 512 * 512].view(-1, 512).any(1).all() and not drows[unused].any()
    half, tiny = (2.0 ** -8 if dtype == BF else 0.0), 2.0 ** -130
    want = dout.double()[:, None] * w.double()[..., None]
    at = slots.clamp(min=0).long()
    within(torch.where(valid[..., None], drows[at], 0.0), torch.where(valid[..., None], want, 0.0), want.abs() * (half + 2.0 ** -23) + tiny)
    terms = torch.where(valid[..., None], rows[at], 0.0).double() * dout.double()[:, None]
    within(dw, terms.sum(-1), terms.abs().sum(-1) * (h / 16 + 64) * 2.0 ** -24 + 2.0 ** -140)
    odd = torch.empty(t * k + 1, dtype=torch.int32, device=DEV)[1:].view(t, k).copy_(slots)
    assert same(ops.moe_ungroup_rows_backward(dout, rows, odd, w), (drows, dw))
    assert torch.equal(ops.moe_ungroup_rows_backward(dout, rows, slots, w, True, False)[0], drows)


def test_gradients_of_many_rows_in_two_graphs():
    """The map of used rows belongs to a call: graphs that are replayed in turn, with other slots each time."""
    g = torch.Generator(device=DEV).manual_seed(6)
    t, k, h = 20000, 8, 24
    m = t * k + 5000
    inputs = [[torch.randn(t, h, device=DEV, generator=g).to(BF), torch.randn(m, h, device=DEV, generator=g).to(BF), many_slots(t, k, m, g), torch.rand(t, k, device=DEV, generator=g)]
              for _ in range(2)]
    ops.moe_ungroup_rows_backward(*inputs[0])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, args in zip(graphs, inputs):
        with torch.cuda.graph(graph):
            outs.append(ops.moe_ungroup_rows_backward(*args))
    for i in range(3):
        for args in inputs:
            args[2].copy_(many_slots(t, k, m, g, 0.3 * i))
        for j in ((0, 1), (1, 0), (0, 1))[i]:
            graphs[j].replay()
        for args, out in zip(inputs, outs):
            assert same(ops.moe_ungroup_rows_backward(*args), out)


def test_gradients_of_many_rows_take_time_like_their_number():
    """Eight times the rows take at most 24 times the time, whatever part of the small case is launches."""
    def milliseconds(t, k, h):
        g = torch.Generator(device=DEV).manual_seed(7)
        m = t * k * 65 // 64 + 100
        args = torch.randn(t, h, device=DEV, generator=g).to(BF), torch.randn(m, h, device=DEV, generator=g).to(BF), many_slots(t, k, m, g), torch.rand(t, k, device=DEV, generator=g)
        times = []
        for _ in range(6):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            ops.moe_ungroup_rows_backward(*args)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)
    assert milliseconds(131072, 8, 16) <= 24 * milliseconds(16384, 8, 16)


def test_rows_past_32_bits():
    t, k, h, e = 40000, 8, 8192, 16
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(t, h, device=DEV, generator=g).to(BF)
    idx = torch.rand(t, e, device=DEV, generator=g).topk(k, -1).indices
    w = torch.rand(t, k, device=DEV, generator=g).requires_grad_()
    x.requires_grad_()
    rows, _, off, slots = ops.moe_group_rows(x, idx, e)
    assert int(off[-1]) == t * k and torch.equal(slots.flatten().sort().values, torch.arange(t * k, device=DEV, dtype=torch.int32))
    for j in (0, k - 1):
        at = slots[:, j].long()
        for i in (0, t - 5):
            assert torch.equal(rows[at[i: i + 5]], x[i: i + 5])
    out = ops.moe_ungroup_rows(rows, slots, w)
    dout = torch.randn(t, h, device=DEV, generator=g).to(BF)
    dx, dw = torch.autograd.grad(out, (x, w), dout)
    i = slice(t - 40, t)
    share = w.detach()[i].double().sum(-1, keepdim=True)
    assert ((out[i].double() - x[i].double() * share).abs() <= (x[i].double() * share).abs() * (2.0 ** -8 + 2.0 ** -20)).all()
    # every row's gradient is rounded, and their sum is
    assert ((dx[i].double() - dout[i].double() * share).abs() <= (dout[i].double() * share).abs() * 2 * (2.0 ** -8 + 2.0 ** -16)).all()
    dots = (x[i].double() * dout[i].double())
    assert ((dw[i].double() - dots.sum(-1, keepdim=True)).abs() <= dots.abs().sum(-1, keepdim=True) * (h / 16 + 64) * 2.0 ** -24).all()


@pytest.mark.parametrize("t,k,e", [(1023, 8, 256), (1024, 8, 256), (1025, 8, 256), (5000, 2, 3), (40000, 8, 1024), (70001, 3, 61), (300000, 1, 2), (9, 32, 1024)])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_sort_of_many_pairs(t, k, e, drop):
    """Against a stable sort: one block, a cluster, uneven experts, pairs of no expert."""
    g = torch.Generator(device=DEV).manual_seed(t)
    idx = (torch.rand(t, k, device=DEV, generator=g) ** 3 * e).long()
    if drop:
        idx = torch.where(torch.rand(t, k, device=DEV, generator=g) < drop, torch.full_like(idx, -1), idx)
    x = torch.arange(t, device=DEV, dtype=torch.float32)[:, None].contiguous()
    rows, _, off, slots = ops.moe_group_rows(x, idx, e)
    key = torch.where(idx < 0, torch.full_like(idx, e), idx).flatten()
    order = key.argsort(stable=True)
    count = torch.bincount(key, minlength=e + 1)[:e]
    n = int(count.sum())
    assert torch.equal(off[1:].long(), count.cumsum(0)) and int(off[0]) == 0
    want = torch.full((t * k,), -1, dtype=torch.int32, device=DEV)
    want[order[:n]] = torch.arange(n, device=DEV, dtype=torch.int32)
    assert torch.equal(slots.flatten(), want)
    assert torch.equal(rows[:n, 0].long(), order[:n] // k) and not rows[n:].any()


def test_group_rows_is_the_order_of_a_dispatch():
    """One rank: the rows that a dispatch hands out, in the same order."""
    from umdk_original_b200 import Buffer, CamConfig
    dev = torch.device("cuda", 0)
    t, h, e, k = 40, 256, 8, 3
    g = torch.Generator().manual_seed(2)
    idx = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(t)]).to(dev)
    x, w = torch.randn(t, h, generator=g).to(dev, BF), torch.rand(t, k, generator=g).to(dev)
    buf = Buffer(None, CamConfig(num_experts=e, max_tokens=t, hidden=h, topk=k, timeout_ms=2000.0), name="order", device=dev, rank=0, num_ranks=1)
    rx, _, _, per_e, _ = ops.moe_dispatch_prefill_quant(x, idx, w, buf.capacity, buf.name, 0, 1, 0)
    rows, _, off, _ = ops.moe_group_rows(x, idx, e)
    assert torch.equal(rows, rx[: t * k]) and torch.equal(off[1:].long(), per_e.cumsum(0).long())
    buf.check()
    buf.destroy()


def test_rows_of_a_dispatch_keep_their_gradients():
    """The rows of a dispatch are overwritten by the next one; what a backward pass reads of them was kept."""
    from umdk_original_b200 import Buffer, CamConfig
    dev = torch.device("cuda", 0)
    t, h = 16, 128
    g = torch.Generator().manual_seed(3)
    idx, one = torch.randint(0, 2, (t, 1), generator=g).to(dev), torch.ones(t, 1, device=dev)
    x = torch.randn(t, h, generator=g).to(dev, BF)
    buf = Buffer(None, CamConfig(num_experts=2, max_tokens=t, hidden=h, topk=1, timeout_ms=2000.0), name="kept", device=dev, rank=0, num_ranks=1)
    rx = ops.moe_dispatch_prefill_quant(x, idx, one, buf.capacity, buf.name, 0, 1, 0)[0][:t]
    rx0, weight = rx.clone(), torch.ones(h, device=dev, dtype=BF, requires_grad=True)
    slots, w = torch.arange(t, device=dev, dtype=torch.int32)[:, None].contiguous(), one.clone().requires_grad_()
    y, out = ops.rms_norm(rx, weight), ops.moe_ungroup_rows(rx, slots, w)
    ops.moe_dispatch_prefill_quant(-2 * x, idx, one, buf.capacity, buf.name, 0, 1, 0)
    assert not torch.equal(rx, rx0)
    ones = torch.ones_like(y)
    got = torch.autograd.grad(y, weight, ones) + torch.autograd.grad(out, w, ones)
    want = torch.autograd.grad(ops.rms_norm(rx0, weight), weight, ones) + torch.autograd.grad(ops.moe_ungroup_rows(rx0, slots, w), w, ones)
    assert same(got, want)
    buf.check()
    buf.destroy()


def test_operands_of_another_device_are_refused():
    c = make()
    for call in (lambda: ops.rms_norm(c["x"], c["weight"].cpu()), lambda: ops.add_rms_norm(c["x"], c["residual"].cpu(), c["weight"]),
                 lambda: ops.moe_route(c["x"], 2, torch.zeros(264)), lambda: ops.moe_group_rows(c["x"], torch.zeros(50, 1, dtype=torch.int64), 2),
                 lambda: ops.moe_ungroup_rows(c["x"], torch.zeros(5, 1, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="device"):
            call()


def test_odd_alignment():
    """Operands that start at any element."""
    c = make(h=264)
    idx = torch.randint(0, 8, (50, 3), device=DEV)

    def shifted(t, n):
        buf = torch.empty(t.numel() + n, device=DEV, dtype=t.dtype)
        return buf[n:].view(t.shape).copy_(t)
    rows, _, off, slots = ops.moe_group_rows(c["x"], idx, 8)
    for n in (1, 2, 4):
        r2, _, off2, slots2 = ops.moe_group_rows(shifted(c["x"], n), idx, 8)
        assert torch.equal(rows, r2) and torch.equal(off, off2) and torch.equal(slots, slots2)
        w = torch.rand(50, 3, device=DEV)
        assert torch.equal(ops.moe_ungroup_rows(rows, slots, w, c["residual"]), ops.moe_ungroup_rows(shifted(rows, n), slots, w, shifted(c["residual"], n)))
        assert torch.equal(ops.moe_route(c["x"], 3)[0], ops.moe_route(shifted(c["x"], n), 3)[0])
    with pytest.raises(RuntimeError, match="aligned"):
        ops.rms_norm_quant(shifted(torch.zeros(4, 128, device=DEV, dtype=BF), 1), torch.ones(128, device=DEV, dtype=BF), 3)
    q8 = torch.randint(-100, 100, (50, 264), device=DEV, dtype=torch.int8)
    assert torch.equal(ops.moe_group_rows(shifted(q8, 3), idx, 8)[0], ops.moe_group_rows(q8, idx, 8)[0])
    want = group64(q8, idx, 8)
    assert torch.equal(ops.moe_group_rows(q8, idx, 8)[0].float(), want[0])


def test_slots_out_of_range_are_left_out():
    rows = torch.randn(6, 40, device=DEV).to(BF).requires_grad_()
    slots = torch.tensor([[0, 6], [2 ** 31 - 1, 3], [-2 ** 31, -1]], device=DEV, dtype=torch.int32)
    w = torch.rand(3, 2, device=DEV).requires_grad_()
    out = ops.moe_ungroup_rows(rows, slots, w)
    inside = ops.moe_ungroup_rows(rows, torch.tensor([[0, -1], [-1, 3], [-1, -1]], device=DEV, dtype=torch.int32), w)
    assert torch.equal(out, inside) and not out[2].any()
    a, b = (torch.autograd.grad(o, (rows, w), torch.ones_like(o)) for o in (out, inside))
    assert same(a, b) and not a[0][[1, 2, 4, 5]].any() and not a[1][2].any()
    none = ops.moe_ungroup_rows(rows[:0].detach(), slots, w)
    assert not none.any()
