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
