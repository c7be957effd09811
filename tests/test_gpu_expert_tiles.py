"""Expert products at sizes where every CTA pair computes several tiles, and the 4-bit forms over clusters, against 64 bits.

Pairs: 74 of them at most on a B200; each case has more than three tiles for every one, of uneven experts (one row, a row less and more
than a block, none), with a K that ends inside a group of scales and result sizes that are no whole tiles in 16 bits."""
import pytest
import torch

from fp4_cases import e4m3_round64, offsets_of, random_fp4, values64
from test_gpu_grouped_mlp import acc, bounds, check, formula64

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROWS = [700, 1, 0, 255, 257, 900, 400, 487]                       # 15 blocks of 256
MORE = [1500, 1, 0, 255, 257, 1100, 600, 900, 511, 700]           # 27


@pytest.fixture(scope="module")
def ops():
    from umdk_original_b200 import ops
    return ops


@pytest.fixture(autouse=True)
def clean(ops):
    from umdk_original_b200.ops import cam_ops
    yield
    torch.cuda.synchronize()
    assert cam_ops.native_module().expert_ops_status()[0] == 0


def product64(a, w, off):
    y = torch.zeros(a.shape[0], w.shape[1], dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(y)
    o = off.tolist()
    for e in range(w.shape[0]):
        r = slice(o[e], o[e + 1])
        y[r], mag[r] = a[r] @ w[e].T, a[r].abs() @ w[e].abs().T
    return y, mag


def acc4(k):
    """Products of two e2m1 values and two scales fit fp32; at most k / 64 additions of partial sums of 64, each rounded or cut to
    2^-23 of the magnitudes at hand, 64 inside them, and two roundings for the global scales."""
    return (k / 64 + 64 + 2) * 2.0 ** -23


def operands(fmt, m, e, k, n, gate):
    """Random codes and scales; with `gate`, scales that keep the sums near 1, where SiLU is neither 0 nor the identity."""
    gen = torch.Generator().manual_seed(m + e + k + n)
    aq, as_ = random_fp4((m, k), fmt, gen)
    wq, ws = random_fp4((e, n, k), fmt, gen)
    ag = wg = None
    if fmt == "nvfp4":  # values have a mean square of 16^2, products of k of them 260 sqrt(k)
        ag = torch.tensor([0.01])
        wg = (0.5 + torch.rand(e, generator=gen)) / (2.6 * k ** 0.5)
    elif gate:          # 8^2 here: 66 sqrt(k)
        down = round(6 + 0.5 * torch.log2(torch.tensor(float(k))).item())
        as_ = (as_.view(torch.uint8) - down).view(torch.float8_e8m0fnu)
    return [None if t is None else t.to(DEV) for t in (aq, as_, wq, ws, ag, wg)]


def loose_rows(m, cnt, head):
    loose = torch.ones(m, dtype=torch.bool, device=DEV)
    loose[head: head + sum(cnt)] = False
    return loose


def check_plain(ops, fmt, cnt, head, tail, k, n):
    m = head + sum(cnt) + tail
    aq, as_, wq, ws, ag, wg = operands(fmt, m, len(cnt), k, n, False)
    off = offsets_of(cnt, head, DEV)
    got = ops.grouped_gemm_fp4(aq, as_, wq, ws, off, ag, wg)
    want, mag = product64(values64(aq, as_, ag), values64(wq, ws, wg), off)
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * acc4(k)).all()
    assert (got[loose_rows(m, cnt, head)] == 0).all()


def check_swiglu(ops, fmt, cnt, head, tail, k, inter):
    """Scales and values against the 64-bit activation; neither bound uses what the kernel returned."""
    m, block = head + sum(cnt) + tail, 16 if fmt == "nvfp4" else 32
    aq, as_, wq, ws, ag, wg = operands(fmt, m, len(cnt), k, 2 * inter, True)
    og = torch.tensor([0.03], device=DEV) if fmt == "nvfp4" else None
    off = offsets_of(cnt, head, DEV)
    q, s = ops.grouped_gemm_fp4_swiglu(aq, as_, wq, ws, off, ag, wg, og)
    gu, mag = product64(values64(aq, as_, ag), values64(wq, ws, wg), off)
    g, u = gu.chunk(2, -1)
    act = g * torch.sigmoid(g) * u
    # accumulated gate and up, |d silu / dg| <= 1.1; SiLU's exponential (21 units of 2^-24 for |g| <= 16), division and two products
    dg, du = (mag * acc4(k)).chunk(2, -1)
    slack = 1.1 * dg * u.abs() + du * (g * torch.sigmoid(g)).abs() + act.abs() * 2.0 ** -19
    live = ~loose_rows(m, cnt, head)
    assert act[live].abs().mean() > 0.05 and g[live].abs().max() < 16  # the inputs are what they are meant to be
    gs = 1.0 if og is None else og.double().item()
    got_s = s.double() if block == 16 else torch.exp2(s.view(torch.uint8).double() - 127)
    amax, asl = (t.unflatten(-1, (-1, block)).abs().amax(-1) for t in (act, slack))
    if block == 16:
        lo, hi = (e4m3_round64(((amax + t * asl) / (6 * gs)).clamp(min=0)) for t in (-1, 1))
    else:
        lo, hi = (torch.exp2(torch.ceil(torch.log2(((amax + t * asl) / 6).clamp(min=2.0 ** -126)))) for t in (-1, 1))
    assert ((got_s >= lo) & (got_s <= hi))[live].all()
    # half a step of e2m1 where the value lies, or what is cut off above 6 d, with either of the scales the interval allows
    a, val = act.abs(), values64(q, s, og)
    half = torch.zeros_like(a)
    for d in (lo, hi):
        dd = (d * gs).repeat_interleave(block, -1)
        half = torch.maximum(half, torch.maximum(dd * torch.where(a <= 2 * dd, 0.25, torch.where(a <= 4 * dd, 0.5, 1.0)), a - 6 * dd))
    assert ((val - act).abs() <= half * (1 + 2.0 ** -20) + slack)[live].all()
    assert (q[~live] == 0).all() and (s.view(torch.uint8)[~live] == 0).all()


# ---------------------------------------------------------------------------- several tiles per pair
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("k,n", [(640, 5120), (2176, 5120), (1280, 4992)])
def test_pairs_product(ops, fmt, k, n, monkeypatch):
    """15 x 20 tiles; 3, 9 and 5 K-blocks, so that a group of four scales is never whole at the end; scales of 1280 values are read in
    wide pieces; 4992 columns end in half a tile."""
    monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    check_plain(ops, fmt, ROWS, 3, 70, k, n)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("k", [640, 2176, 1280])
def test_pairs_swiglu(ops, fmt, k, monkeypatch):
    monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    check_swiglu(ops, fmt, ROWS, 3, 70, k, 2560)  # 15 x 20 tiles


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pairs_forward_and_gradients(ops, dtype, monkeypatch):
    """up 27 x 11 tiles, down and dx 27 x 9, dact 27 x 11."""
    monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    h, inter, head, tail = 4104, 2568, 5, 90
    gen = torch.Generator(device=DEV).manual_seed(31)
    e, m = len(MORE), head + sum(MORE) + tail
    x = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    w1 = (torch.randn(e, 2 * inter, h, device=DEV, generator=gen) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, inter, device=DEV, generator=gen) * inter ** -0.5).to(dtype)
    dy = torch.randn(m, h, device=DEV, generator=gen).to(dtype)
    off = offsets_of(MORE, head, DEV)
    half, tiny = bounds(dtype)
    want, tol = formula64(x, w1, w2, dy, off, half, acc)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    y = ops.grouped_mlp(*leaves, off)
    with torch.no_grad():
        assert torch.equal(ops.grouped_mlp(x, w1, w2, off), y)
    dx, dw1, dw2 = torch.autograd.grad(y, leaves, dy)
    check({"y": y.detach(), "dx": dx, "dw1": dw1, "dw2": dw2}, want, tol, tiny * (m + 2 * inter + h))
    loose = loose_rows(m, MORE, head)
    assert (y[loose] == 0).all() and (dx[loose] == 0).all() and (dw1[2] == 0).all() and (dw2[2] == 0).all()


# ---------------------------------------------------------------------------- 4 bits over clusters
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("split", ["1", "2", "4"])
@pytest.mark.parametrize("cnt,k", [([10, 0, 29, 1], 4096), ([450, 450], 4096), ([33, 128, 139], 5248)])  # 4, 4 and 6 groups of K-blocks
@pytest.mark.parametrize("swiglu", [False, True])
def test_clusters(ops, fmt, split, cnt, k, swiglu, monkeypatch):
    """A tile's K-blocks divided among 1, 2 and 4 CTAs (37 clusters of 4), several tiles per cluster at 900 rows."""
    monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "1")
    monkeypatch.setenv("UMDK_CAM_EXPERT_SPLIT", split)
    if swiglu:
        check_swiglu(ops, fmt, cnt, 1, 2, k, 1024)
    else:
        check_plain(ops, fmt, cnt, 1, 2, k, 1024)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("cnt,k,inter", [([1] * 8, 7168, 2048), ([3, 0, 20, 9] * 4, 4096, 1024), ([60] * 8, 2048, 512), ([160], 4096, 1024)])
def test_chosen_form_swiglu(ops, fmt, cnt, k, inter):
    """The form and the split that the rule takes for few rows."""
    check_swiglu(ops, fmt, cnt, 0, 5, k, inter)


def test_gradient_at_an_odd_offset(ops):
    """The gradient that autograd hands over is a slice of another one's memory, two bytes past a 16-byte boundary."""
    m, h, inter = 40, 64, 32
    gen = torch.Generator(device=DEV).manual_seed(41)
    x = torch.randn(m, h, device=DEV, generator=gen).to(torch.bfloat16)
    leaves = [x.requires_grad_(), *[(torch.randn(*s, device=DEV, generator=gen) / 8).to(torch.bfloat16).requires_grad_() for s in ((2, 2 * inter, h), (2, h, inter))]]
    off = offsets_of([17, 23], device=DEV)
    dy = torch.randn(m * h + 1, device=DEV, generator=gen).to(torch.bfloat16)
    y = ops.grouped_mlp(*leaves, off)
    got = torch.autograd.grad(torch.cat([y.new_zeros(1), y.flatten()]), leaves, dy, retain_graph=True)
    want = torch.autograd.grad(y, leaves, dy[1:].view(m, h).clone())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
