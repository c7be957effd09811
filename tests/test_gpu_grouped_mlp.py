"""Gated feed-forward block of 16-bit experts on the GPU: outputs and gradients against the formula in 64 bits."""
import pytest
import torch

from fp4_cases import offsets_of

pytestmark = pytest.mark.gpu

DEV = "cuda"
# rows per expert, rows before the first, rows after the last
COUNTS = {
    "one row": ([1], 0, 0),
    "one expert, 300 rows": ([300], 0, 0),
    "holes": ([0, 3, 0, 0, 70, 1, 0], 0, 5),
    "block borders": ([63, 64, 65, 128, 255, 256, 257], 0, 0),
    "head and tail": ([40, 0, 200], 7, 260),
    "no rows at all": ([0, 0], 0, 9),
}


@pytest.fixture(scope="module")
def ops():
    from umdk_original_b200 import ops
    return ops


def make(dtype, h, inter, counts, seed=0):
    cnt, head, tail = COUNTS[counts]
    gen = torch.Generator(device=DEV).manual_seed(seed + h + inter)
    e, m = len(cnt), head + sum(cnt) + tail
    x = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    w1 = (torch.randn(e, 2 * inter, h, device=DEV, generator=gen) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, inter, device=DEV, generator=gen) * inter ** -0.5).to(dtype)
    dy = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    return x, w1, w2, dy, offsets_of(cnt, head, DEV)


def sums64(a, b):
    """(a @ b, sum of magnitudes)."""
    return a @ b, a.abs() @ b.abs()


def formula64(x, w1, w2, dy, off, half, acc):
    """Values in fp64 and bounds for what fp32 accumulators (`acc(k)` of the magnitudes of a sum of k terms) and one rounding of
    act and of dgu to 16 bits (`half` a step relative) may do to them."""
    x, w1, w2, dy = (t.double() for t in (x, w1, w2, dy))
    m, h, e, i = x.shape[0], x.shape[1], w1.shape[0], w2.shape[2]
    z = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.float64)  # noqa: E731
    out = {k: z(*s) for k, s in dict(y=(m, h), dx=(m, h), dw1=(e, 2 * i, h), dw2=(e, h, i)).items()}
    tol = {k: v.clone() for k, v in out.items()}
    o = off.tolist()
    for j in range(e):
        a, b = o[j], o[j + 1]
        if a == b:
            continue
        r = slice(a, b)
        gu, gum = sums64(x[r], w1[j].T)
        g, u = gu.chunk(2, -1)
        eg, eu = (gum * acc(h)).chunk(2, -1)
        s = torch.sigmoid(g)
        silu, dsilu = g * s, s * (1 + g * (1 - s))
        # |silu'| <= 1.1, |silu''| <= 0.5; a few fp32 operations (expf, division, products): 2^-20 of the value
        act = silu * u
        eact = 1.1 * eg * u.abs() + silu.abs() * eu + act.abs() * (half + 2.0 ** -20)
        out["y"][r], ym = sums64(act, w2[j].T)
        tol["y"][r] = eact @ w2[j].abs().T + ym * acc(i)
        da, dam = sums64(dy[r], w2[j])
        eda = dam * acc(h)
        dg, du = da * u * dsilu, da * silu
        edg = eda * (u * dsilu).abs() + da.abs() * (eu * dsilu.abs() + u.abs() * 0.5 * eg) + da.abs() * u.abs() * 2.0 ** -20 + dg.abs() * half
        edu = eda * silu.abs() + da.abs() * 1.1 * eg + du.abs() * (half + 2.0 ** -20)
        dgu, edgu = torch.cat([dg, du], -1), torch.cat([edg, edu], -1)
        out["dx"][r], mag = sums64(dgu, w1[j])
        tol["dx"][r] = edgu @ w1[j].abs() + mag * acc(2 * i)
        out["dw1"][j], mag = sums64(dgu.T, x[r])
        tol["dw1"][j] = edgu.T @ x[r].abs() + mag * acc(b - a)
        out["dw2"][j], mag = sums64(dy[r].T, act)
        tol["dw2"][j] = dy[r].abs().T @ eact + mag * acc(b - a)
    for k in out:
        tol[k] += out[k].abs() * half
    return out, tol


def acc(k):
    """Sums of k products in fp32: the products of two 16-bit values are exact; at most k / 16 + 16 roundings or cuts of 2^-23."""
    return (k / 16 + 17) * 2.0 ** -23


def bounds(dtype):
    # half a step; fp16 also has subnormals, whose half step is 2^-25
    return torch.finfo(dtype).eps / 2, (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check(got, want, tol, tiny, scale=1.0):
    for k, v in got.items():
        bad = (v.double() - want[k]).abs() > tol[k] + tiny * scale
        assert not bad.any(), (k, int(bad.sum()), float(((v.double() - want[k]).abs() / (tol[k] + 1e-30)).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,inter", [(8, 8), (136, 72), (256, 128), (1000, 344), (512, 640)])
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("form", ["chosen", "pairs"])
def test_forward_and_gradients(ops, dtype, h, inter, counts, form, monkeypatch):
    if form == "pairs":  # the form for many rows per expert, at all sizes
        monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    x, w1, w2, dy, off = make(dtype, h, inter, counts)
    half, tiny = bounds(dtype)
    want, tol = formula64(x, w1, w2, dy, off, half, acc)
    with torch.no_grad():
        y0 = ops.grouped_mlp(x, w1, w2, off)
    check({"y": y0}, want, tol, tiny * (inter + 1))
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    assert torch.equal(y, y0)
    dx, dw1, dw2 = torch.autograd.grad(y, leaves, dy)
    check({"dx": dx, "dw1": dw1, "dw2": dw2}, want, tol, tiny * (x.shape[0] + 2 * inter + h))
    cnt, head, _ = COUNTS[counts]
    loose = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    loose[head: head + sum(cnt)] = False
    assert (y[loose] == 0).all() and (dx[loose] == 0).all()
    for e, c in enumerate(cnt):
        if c == 0:
            assert (dw1[e] == 0).all() and (dw2[e] == 0).all()


def test_status_is_clean(ops):
    from umdk_original_b200.ops import cam_ops
    assert cam_ops.native_module().expert_ops_status()[0] == 0


@pytest.mark.parametrize("m,e,h,inter", [(1, 1, 512, 256), (3, 2, 4096, 64), (40, 8, 264, 1024), (640, 1, 1024, 256), (130, 1, 2048, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows(ops, dtype, m, e, h, inter):
    """Sizes at which the form for few rows divides a product among several CTAs, or has room for 32, 64 or 128 rows."""
    gen = torch.Generator(device=DEV).manual_seed(m + h)
    x = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    w1 = (torch.randn(e, 2 * inter, h, device=DEV, generator=gen) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, inter, device=DEV, generator=gen) * inter ** -0.5).to(dtype)
    dy = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    cnt = torch.bincount(torch.randint(0, e, (m,), generator=torch.Generator().manual_seed(m)), minlength=e).tolist()
    off = offsets_of(cnt, 0, DEV)
    half, tiny = bounds(dtype)
    want, tol = formula64(x, w1, w2, dy, off, half, acc)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    dx, dw1, dw2 = torch.autograd.grad(y, leaves, dy)
    check({"y": y.detach(), "dx": dx, "dw1": dw1, "dw2": dw2}, want, tol, tiny * (m + 2 * inter + h))


@pytest.mark.parametrize("split", ["1", "2", "4"])
@pytest.mark.parametrize("m,e,h,inter", [(33, 2, 1032, 520), (700, 3, 640, 328), (1300, 1, 2048, 512)])
def test_tiles_shared_by_a_cluster(ops, split, m, e, h, inter, monkeypatch):
    """The form for few rows at any number of rows, with 1, 2 and 4 CTAs per tile and several tiles per cluster."""
    monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "1")
    monkeypatch.setenv("UMDK_CAM_EXPERT_SPLIT", split)
    test_few_rows(ops, torch.bfloat16, m, e, h, inter)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,inter", [(8, 8), (264, 136), (4104, 520)])
@pytest.mark.parametrize("cnt,head,tail", [([1], 0, 0), ([2], 0, 0), ([0, 1, 0, 1], 0, 0), ([3], 0, 0), ([0, 1, 0], 1, 1), ([5, 0, 2], 2, 3), ([16], 0, 0),
                                           ([0, 0], 0, 2)])
def test_a_handful_of_rows(ops, dtype, h, inter, cnt, head, tail):
    """The form on the ordinary cores: one, two and more rows, several blocks of rows, rows of no expert, a NaN in an idle expert."""
    gen = torch.Generator(device=DEV).manual_seed(h + sum(cnt))
    e, m = len(cnt), head + sum(cnt) + tail
    x = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    w1 = (torch.randn(e, 2 * inter, h, device=DEV, generator=gen) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, inter, device=DEV, generator=gen) * inter ** -0.5).to(dtype)
    dy = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    off = offsets_of(cnt, head, DEV)
    half, tiny = bounds(dtype)
    want, tol = formula64(x, w1, w2, dy, off, half, acc)
    for j in range(e):
        if cnt[j] == 0:
            w1[j], w2[j] = float("nan"), float("nan")
    x[:head], x[m - tail:] = float("nan"), float("nan")
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    with torch.no_grad():
        assert torch.equal(ops.grouped_mlp(x, w1, w2, off), y)
    dx, dw1, dw2 = torch.autograd.grad(y, leaves, dy)
    check({"y": y.detach(), "dx": dx, "dw1": dw1, "dw2": dw2}, want, tol, tiny * (m + 2 * inter + h))


def test_two_runs_give_the_same_bits(ops):
    x, w1, w2, dy, off = make(torch.bfloat16, 1000, 344, "block borders")
    runs = []
    for _ in range(2):
        leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
        y = ops.grouped_mlp(*leaves, off)
        runs.append((y, *torch.autograd.grad(y, leaves, dy)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("form", ["chosen", "pairs"])
def test_nan_stays_with_its_expert(ops, form, monkeypatch):
    """Rows and weights of one expert, and rows of none, are NaN and infinities; the others' results are as without them."""
    if form == "pairs":
        monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    x, w1, w2, dy, off = make(torch.bfloat16, 136, 72, "head and tail")  # experts of 40, 0 and 200 rows behind 7 and before 260
    cnt = [40, 100, 100]
    off = offsets_of(cnt, 7, DEV)
    clean = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y0 = ops.grouped_mlp(*clean, off)
    g0 = torch.autograd.grad(y0, clean, dy)
    bad = [t.clone() for t in (x, w1, w2, dy)]
    bad[0][:7], bad[0][247:], bad[0][47:147] = float("nan"), float("inf"), float("nan")
    bad[1][1], bad[2][1] = float("nan"), float("inf")
    bad[3][:7], bad[3][247:], bad[3][47:147] = float("inf"), float("nan"), float("-inf")
    leaves = [t.requires_grad_() for t in bad[:3]]
    y = ops.grouped_mlp(*leaves, off)
    g = torch.autograd.grad(y, leaves, bad[3])
    keep = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    keep[47:147] = False
    assert torch.equal(y[keep], y0[keep]) and torch.equal(g[0][keep], g0[0][keep])
    for i in (1, 2):
        assert torch.equal(g[i][0], g0[i][0]) and torch.equal(g[i][2], g0[i][2])
        assert not g[i][1].isfinite().all()


def test_offsets_past_32_bits(ops):
    """Weights of more than 2^32 bytes: the last expert's."""
    e, h, inter = 66, 8192, 2048
    gen = torch.Generator(device=DEV).manual_seed(5)
    w1 = torch.empty(e, 2 * inter, h, device=DEV, dtype=torch.bfloat16)
    w2 = torch.empty(e, h, inter, device=DEV, dtype=torch.bfloat16)
    assert w1.numel() * 2 > 2 ** 32
    w1[-1] = torch.randn(2 * inter, h, device=DEV, generator=gen) * h ** -0.5
    w2[-1] = torch.randn(h, inter, device=DEV, generator=gen) * inter ** -0.5
    x = torch.randn(70, h, device=DEV, generator=gen).to(torch.bfloat16)
    dy = torch.randn(70, h, device=DEV, generator=gen).to(torch.bfloat16)
    off = torch.tensor([0] * e + [70], dtype=torch.int32, device=DEV)
    want, tol = formula64(x, w1[-1:], w2[-1:], dy, torch.tensor([0, 70]), *[bounds(torch.bfloat16)[0], acc])
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    dx, dw1, dw2 = torch.autograd.grad(y, leaves, dy)
    check({"y": y.detach(), "dx": dx, "dw1": dw1[-1:], "dw2": dw2[-1:]}, want, tol, 0.0)
    assert (dw1[:-1] == 0).all() and (dw2[:-1] == 0).all()


def test_wild_offsets_stay_inside(ops):
    """Offsets that make no sense (decreasing, negative, past the rows) are clamped; what they select is computed, nothing else is
    touched and no wait runs out."""
    from umdk_original_b200.ops import cam_ops
    x, w1, w2, dy, _ = make(torch.bfloat16, 136, 72, "holes")
    for off in ([5, -3, 2 ** 31 - 1, 7, 7, 0, 10, 3], [0, 0, 0, 0, 0, 0, 0, 10 ** 9], [79, 79, 79, 79, 79, 79, 79, -5]):
        o = torch.tensor(off, dtype=torch.int32, device=DEV)
        leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
        y = ops.grouped_mlp(*leaves, o)
        torch.autograd.grad(y, leaves, dy)
        torch.cuda.synchronize()
        assert cam_ops.native_module().expert_ops_status()[0] == 0


def test_capture_and_replay(ops):
    """Forward and backward in one CUDA graph, replayed with other rows, weights and offsets; and a side stream."""
    x, w1, w2, dy, off = make(torch.bfloat16, 256, 128, "holes")
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    d, o = dy.clone(), off.clone()

    def step():
        y = ops.grouped_mlp(*leaves, o)
        return (y.detach(), *torch.autograd.grad(y, leaves, d))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(first, want))
    del first
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x2, w12, w22, dy2, _ = make(torch.bfloat16, 256, 128, "holes", seed=9)
    with torch.no_grad():
        for a, b in zip(leaves, (x2, w12, w22)):
            a.copy_(b)
    d.copy_(dy2)
    o.copy_(offsets_of([10, 0, 0, 30, 1, 2, 3], 2, DEV))
    g.replay()
    got = [t.clone() for t in out]
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_capture_beside_an_eager_graph_is_refused(ops):
    x, w1, w2, dy, off = make(torch.bfloat16, 256, 128, "holes")
    w1.requires_grad_()
    eager = ops.grouped_mlp(x, w1, w2, off)  # holds w1's accumulation node
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go of its outputs"):
        with torch.cuda.graph(g):
            ops.grouped_mlp(x, w1, w2, off)
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.grouped_mlp(x, w1, w2, off)
        dw, = torch.autograd.grad(y, w1, dy)
    g.replay()
    y2 = ops.grouped_mlp(x, w1, w2, off)
    assert torch.equal(y, y2) and torch.equal(dw, torch.autograd.grad(y2, w1, dy)[0])


def test_refusals(ops):
    from test_grouped_mlp_cpu import refusals
    for call in refusals(DEV):
        with pytest.raises(RuntimeError, match="umdk_cam_op_lib"):
            call()
    x, w1, w2, dy, off = make(torch.bfloat16, 256, 128, "holes")
    with pytest.raises(RuntimeError, match="device"):
        ops.grouped_mlp(x, w1, w2, off.cpu())
    shifted = torch.empty(x.numel() + 1, device=DEV, dtype=x.dtype)[1:].view_as(x)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.grouped_mlp(shifted, w1, w2, off)


def test_training_with_accumulated_gradients(ops):
    """.backward() twice accumulates; gradients of an expanded scalar; weights that do not want a gradient."""
    x, w1, w2, dy, off = make(torch.float16, 136, 72, "block borders")
    w1.requires_grad_()
    ops.grouped_mlp(x, w1, w2, off).float().sum().backward()
    once = w1.grad.clone()
    ops.grouped_mlp(x, w1, w2, off).float().sum().backward()
    assert torch.equal(w1.grad, (once.float() * 2).half())


@pytest.mark.parametrize("fmt", ["bf16", "nvfp4", "mxfp4"])
def test_dispatch_experts_combine(ops, fmt):
    """The operators as they are used: rows from a dispatch, the experts' MLP, the weighted sum of the combine."""
    from umdk_original_b200 import Buffer, CamConfig
    from umdk_original_b200.models import ExpertMLP, offsets_from_counts
    t, h, inter, e, k = 64, 256, 128, 8, 2
    gen = torch.Generator().manual_seed(7)
    x = torch.randn(t, h, generator=gen).to(torch.bfloat16).to(DEV)
    idx = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)]).to(DEV)
    wt = torch.rand(t, k, generator=gen).to(DEV)
    buf = Buffer(None, CamConfig(num_experts=e, max_tokens=t, hidden=h, topk=k, timeout_ms=2000.0), name="expert_mlp_" + fmt,
                 device=torch.device(DEV, 0), rank=0, num_ranks=1)
    mlp = ExpertMLP(e, h, inter, device=DEV, seed=1)
    layer = mlp if fmt == "bf16" else mlp.quantized(fmt)
    with torch.no_grad():
        # a receive buffer of fixed size: rows past the last expert belong to none
        rx, src, cnt, per_e, _ = ops.moe_dispatch_prefill_quant(x, idx, wt, buf.capacity, buf.name, 0, 1, 0)
        off = offsets_from_counts(per_e)
        y = layer(rx, off)
        out = ops.moe_combine_prefill(y, idx, wt, src, cnt, buf.name, 0, 1)
    buf.check()
    if fmt == "bf16":
        w1, w2 = mlp.w1.detach().double(), mlp.w2.detach().double()
    else:
        w1 = ops.dequantize_fp4(layer.w1_q, layer.w1_s, layer.w1_gs, torch.float32).double()
        w2 = ops.dequantize_fp4(layer.w2_q, layer.w2_s, layer.w2_gs, torch.float32).double()

    def rows64(v):
        if fmt == "bf16":
            return v
        q, s = ops.quantize_fp4(v.float().contiguous(), layer.block)
        return ops.dequantize_fp4(q, s, None, torch.float32).double()
    want = torch.zeros(t, h, dtype=torch.float64, device=DEV)
    for j in range(k):
        g, u = torch.einsum("th,tih->ti", rows64(x.double()), w1[idx[:, j]]).chunk(2, -1)
        act = rows64(g * torch.sigmoid(g) * u)
        want += torch.einsum("ti,thi->th", act, w2[idx[:, j]]) * wt[:, j: j + 1].double()
    # bf16: act, expert output and result are rounded (half a step, 2^-8, each); 4 bits: a value of act near the middle between two
    # points may round to the other one, which moves few values by a third at most
    err = (out.double() - want).norm() / want.norm()
    assert err < (3 * 2.0 ** -8 if fmt == "bf16" else 0.02)
    if fmt == "bf16":
        y = mlp(rx.clone(), off)
        dw1, dw2 = torch.autograd.grad(y.float().square().sum(), (mlp.w1, mlp.w2))
        assert dw1.isfinite().all() and dw2.isfinite().all() and dw1.abs().sum() > 0
    buf.destroy()


def test_backward_after_the_next_dispatch(ops):
    """Two layers share a Buffer: the second dispatch overwrites the rows that the first layer's experts saw, before backward runs."""
    from umdk_original_b200 import Buffer, CamConfig
    from umdk_original_b200.models import ExpertMLP, offsets_from_counts
    t, h, inter, e, k = 32, 128, 64, 4, 2
    gen = torch.Generator().manual_seed(11)
    idx = torch.stack([torch.randperm(e, generator=gen)[:k] for _ in range(t)]).to(DEV)
    wt = torch.rand(t, k, generator=gen).to(DEV)
    buf = Buffer(None, CamConfig(num_experts=e, max_tokens=t, hidden=h, topk=k, timeout_ms=2000.0), name="expert_mlp_two_layers",
                 device=torch.device(DEV, 0), rank=0, num_ranks=1)
    layers = [ExpertMLP(e, h, inter, device=DEV, seed=s) for s in (1, 2)]
    loss, rows = 0.0, []
    for layer in layers:
        x = torch.randn(t, h, generator=gen).to(torch.bfloat16).to(DEV)
        rx, _, _, per_e, _ = ops.moe_dispatch_prefill_quant(x, idx, wt, buf.capacity, buf.name, 0, 1, 0)
        off = offsets_from_counts(per_e)
        rows.append((rx, rx.clone(), off))
        loss = loss + layer(rx, off).float().square().sum()
    assert not torch.equal(rows[0][0], rows[0][1])  # overwritten
    got = torch.autograd.grad(loss, [p for layer in layers for p in (layer.w1, layer.w2)])
    want = []
    for layer, (_, rx, off) in zip(layers, rows):
        want += torch.autograd.grad(layer(rx, off).float().square().sum(), (layer.w1, layer.w2))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf.check()
    buf.destroy()


def test_waits_for_another_stream(ops):
    """The kernels may start before the one ahead of them on their stream has finished, but not before an event they wait for."""
    x, w1, w2, dy, off = make(torch.bfloat16, 256, 128, "holes")
    want = ops.grouped_mlp(x, w1, w2, off)
    late = torch.zeros_like(w1)
    side = torch.cuda.Stream()

    def run():
        side.wait_stream(torch.cuda.current_stream())
        y = ops.grouped_mlp(x, w1, w2, off)  # the kernel ahead on this stream
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)  # about a millisecond
            late.copy_(w1)
        torch.cuda.current_stream().wait_stream(side)
        return y, ops.grouped_mlp(x, late, w2, off)

    assert all(torch.equal(y, want) for y in run())
    late.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    late.zero_()
    g.replay()
    assert all(torch.equal(y, want) for y in out)


def test_calls_from_two_host_threads(ops):
    import threading
    x, w1, w2, dy, off = make(torch.bfloat16, 264, 136, "holes")
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
            for _ in range(20):
                y = ops.grouped_mlp(*leaves, off)
                got[i] = (y.detach(), *torch.autograd.grad(y, leaves, dy))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    want = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_status_after_everything(ops):
    from umdk_original_b200.ops import cam_ops
    assert cam_ops.native_module().expert_ops_status()[0] == 0
