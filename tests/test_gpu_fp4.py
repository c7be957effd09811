"""4-bit operators on the GPU against their definitions in 64 bits."""
import pytest
import torch

from fp4_cases import e4m3_round64, offsets_of, quantise64, random_fp4, values64

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from umdk_original_b200 import ops
    return ops


# ---------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,g", [(16, None), (16, 2.0 ** -7), (16, 0.0123), (32, None)])
@pytest.mark.parametrize("shape", [(1, 32), (1, 7168), (3, 160), (127, 4096), (5, 2, 96)])
def test_quantise_bits(ops, dtype, block, g, shape):
    """Codes and scales are the definition's: a quotient of a 16-bit value and a 4-bit scale is either a tie or far from one."""
    gen = torch.Generator().manual_seed(hash((block, shape)) % 1000)
    x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape[-1], generator=gen))
    x[..., :block] = 0  # a block of zeros
    x = x.to(dtype)
    gs = None if g is None else torch.tensor([g])
    q, s = ops.quantize_fp4(x.to(DEV), block, None if gs is None else gs.to(DEV))
    assert q.shape == (*shape[:-1], shape[-1] // 2) and s.shape == (*shape[:-1], shape[-1] // block)
    want_q, want_s = quantise64(x, block, gs)
    got_s = s.cpu().double() if block == 16 else torch.exp2(s.cpu().view(torch.uint8).double() - 127)
    assert torch.equal(got_s, want_s)
    got_q = values64(q.cpu(), torch.ones(*shape[:-1], 1).to(torch.float8_e4m3fn))
    assert torch.equal(got_q, want_q)


def test_quantise_ties_and_saturation(ops):
    """Every half-way point with a scale that is not a power of two, both signs; values above 6 s after the scale was rounded down."""
    pts = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for scale in (1.0, 1.125, 1.625, 0.6875):
        x = torch.cat([pts * scale, -pts * scale]).reshape(1, 16)
        assert torch.equal(x.to(torch.bfloat16).float(), x)
        q, s = ops.quantize_fp4(x.to(DEV, torch.bfloat16), 16)
        assert float(s.cpu().double()) == scale
        want = torch.tensor([0, 1, 1, 2, 2, 4, 4, 6.0]).double()
        got = values64(q.cpu(), torch.ones(1, 1).to(torch.float8_e4m3fn))[0]
        assert torch.equal(got, torch.cat([want, -want]))
    x = torch.full((1, 16), 6.19)  # amax / 6 = 1.03 -> scale 1.0, quotient 6.19 -> 6
    q, s = ops.quantize_fp4(x.to(DEV, torch.bfloat16), 16)
    assert float(s.cpu().double()) == 1.0 and torch.equal(ops.dequantize_fp4(q, s).cpu().float(), torch.full((1, 16), 6.0))


@pytest.mark.parametrize("block", [16, 32])
def test_quantise_infinities_and_nan_stay_in_their_block(ops, block):
    x = torch.randn(1, 4 * block, generator=torch.Generator().manual_seed(3))
    x[0, 3] = float("inf")
    x[0, block + 1] = float("-inf")
    x[0, 2 * block + 5] = float("nan")
    q, s = ops.quantize_fp4(x.to(DEV), block)
    v = ops.dequantize_fp4(q, s, dtype=torch.float32).cpu()[0]
    top = 6 * (448.0 if block == 16 else 2.0 ** 127)
    if block == 16:
        assert v[3] == top and v[block + 1] == -top
    else:
        assert v[3] == float("inf") and v[block + 1] == float("-inf")  # 6 x 2^127
    assert v[2 * block: 3 * block].isnan().all()
    assert not v[: 2 * block].isnan().any() and not v[3 * block:].isnan().any()
    want, _ = quantise64(x[:, 3 * block:], block)
    assert torch.equal(values64(q.cpu()[:, 3 * block // 2:], torch.ones(1, 1).to(torch.float8_e4m3fn)), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_dequantise(ops, dtype, fmt):
    gen = torch.Generator().manual_seed(5)
    q, s = random_fp4((3, 17, 96), fmt, gen)
    gs = torch.rand(3, generator=gen) + 0.5 if fmt == "nvfp4" else None
    got = ops.dequantize_fp4(q.to(DEV), s.to(DEV), None if gs is None else gs.to(DEV), dtype).cpu()
    # fp32: scale x global scale and value x scale round once each; then the output type's own half step
    want = values64(q, s, gs)
    assert got.dtype == dtype
    assert ((got.double() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -23)).all()


def test_expert_scales_and_empty(ops):
    gen = torch.Generator().manual_seed(6)
    w = torch.randn(4, 24, 64, generator=gen).to(torch.bfloat16)
    gs = torch.tensor([2.0 ** -6, 2.0 ** -8, 1.0, 2.0 ** -3])
    q, s = ops.quantize_fp4(w.to(DEV), 16, gs.to(DEV))
    want_q, want_s = quantise64(w, 16, gs)
    assert torch.equal(s.cpu().double(), want_s)
    assert torch.equal(values64(q.cpu(), torch.ones(4, 24, 1).to(torch.float8_e4m3fn)), want_q)
    q, s = ops.quantize_fp4(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16), 32)
    assert q.shape == (0, 32) and s.shape == (0, 2) and ops.dequantize_fp4(q, s).shape == (0, 64)


# ---------------------------------------------------------------------------- products
COUNTS = {
    "one row": ([1], 0, 0),
    "one expert, 129 rows": ([129], 0, 0),
    "holes": ([0, 3, 0, 0, 70, 1, 0], 0, 5),
    "tile borders": ([32, 33, 96, 97, 128, 255, 256, 257], 0, 0),
    "head and tail": ([40, 0, 200], 7, 260),
    "no rows at all": ([0, 0], 0, 9),
}


def _gs(fmt, e, gen):
    if fmt == "mxfp4":
        return None, None
    return torch.rand(1, generator=gen) * 0.1, torch.rand(e, generator=gen) * 0.1


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _product64(a, w, off, m):
    """(product, sum of magnitudes) per expert in fp64."""
    y = torch.zeros(m, w.shape[1], dtype=torch.float64, device=a.device)
    mag = torch.zeros_like(y)
    o = off.tolist()
    for e in range(w.shape[0]):
        y[o[e]: o[e + 1]] = a[o[e]: o[e + 1]] @ w[e].T
        mag[o[e]: o[e + 1]] = a[o[e]: o[e + 1]].abs() @ w[e].abs().T
    return y, mag


def _acc_tol(k):
    """Products of two e2m1 values and two scales fit fp32 exactly; at most k / 64 additions of partial sums of 64, each rounded or
    cut to 2^-23 of the magnitudes at hand, and one more for the global scales."""
    return (k / 64 + 64 + 2) * 2.0 ** -23


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("k,n", [(128, 128), (384, 256), (512, 640), (2048, 384)])
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("form", ["chosen", "pairs"])
def test_product(ops, fmt, k, n, counts, form, monkeypatch):
    if form == "pairs":  # the form for many rows per expert, at all sizes
        monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    cnt, head, tail = COUNTS[counts]
    gen = torch.Generator().manual_seed(k + n)
    e, m = len(cnt), head + sum(cnt) + tail
    aq, as_ = random_fp4((m, k), fmt, gen)
    wq, ws = random_fp4((e, n, k), fmt, gen)
    ag, wg = _gs(fmt, e, gen)
    off = offsets_of(cnt, head)
    got = ops.grouped_gemm_fp4(*_dev(aq, as_, wq, ws, off, ag, wg))
    want, mag = _product64(values64(*_dev(aq, as_, ag)), values64(*_dev(wq, ws, wg)), off, m)
    assert got.dtype == torch.bfloat16 and got.shape == (m, n)
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * _acc_tol(k)).all()
    loose = torch.ones(m, dtype=torch.bool)
    loose[head: head + sum(cnt)] = False
    assert (got.cpu()[loose] == 0).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("k,inter", [(128, 128), (384, 256), (1024, 384)])
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("form", ["chosen", "pairs"])
def test_swiglu(ops, fmt, k, inter, counts, form, monkeypatch):
    if form == "pairs":
        monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "0")
    cnt, head, tail = COUNTS[counts]
    block = 16 if fmt == "nvfp4" else 32
    gen = torch.Generator().manual_seed(k + inter)
    e, m = len(cnt), head + sum(cnt) + tail
    aq, as_ = random_fp4((m, k), fmt, gen)
    wq, ws = random_fp4((e, 2 * inter, k), fmt, gen)
    if fmt == "nvfp4":
        ag, wg, og = torch.full((1,), 0.02), torch.rand(e, generator=gen) * 0.01, torch.full((1,), 0.03)
    else:  # keep gates in the range where SiLU is neither 0 nor the identity
        ag = wg = og = None
        as_ = (as_.view(torch.uint8) - 9).view(torch.float8_e8m0fnu)
    off = offsets_of(cnt, head)
    q, s = ops.grouped_gemm_fp4_swiglu(*_dev(aq, as_, wq, ws, off, ag, wg, og))
    gu, mag = _product64(values64(*_dev(aq, as_, ag)), values64(*_dev(wq, ws, wg)), off, m)
    g, u = gu.chunk(2, -1)
    act = g * torch.sigmoid(g) * u
    # fp32: accumulated gate and up, then SiLU's exponential, division and two products (a few units of 2^-23 of the value;
    # |d silu / dg| <= 1.1)
    dg, du = (mag * _acc_tol(k)).chunk(2, -1)
    slack = 1.1 * dg * u.abs() + du * (g * torch.sigmoid(g)).abs() + act.abs() * 2.0 ** -19
    live = torch.zeros(m, dtype=torch.bool, device=DEV)
    live[head: head + sum(cnt)] = True
    got_s = s.double() if block == 16 else torch.exp2(s.view(torch.uint8).double() - 127)
    d = got_s * (1.0 if og is None else og.double().item())
    amax = act.unflatten(-1, (-1, block)).abs().amax(-1)
    asl = slack.unflatten(-1, (-1, block)).amax(-1)
    if block == 16:
        lo, hi = (e4m3_round64(((amax + t * asl) / (6 * og.double().item())).clamp(min=0)) for t in (-1, 1))
        assert ((got_s >= lo) & (got_s <= hi))[live].all()
    else:
        lo, hi = (torch.exp2(torch.ceil(torch.log2(((amax + t * asl) / 6).clamp(min=2.0 ** -126)))) for t in (-1, 1))
        ok = ((got_s >= lo) & (got_s <= hi)) | (amax <= asl)
        assert ok[live].all()
    val = values64(q, s, None if og is None else og.to(DEV))
    dd = d.repeat_interleave(block, -1)
    a = act.abs()
    # Half a step of e2m1 where the value lies, or what is cut off above 6 d.  The scale is rounded to nearest, so amax / d may
    # exceed 6: by 1/16 for a normal e4m3, but a scale that rounds to the smallest subnormal, 2^-9, stands for up to 1.5 x 2^-9
    # (amax / d up to 9).
    half = torch.maximum(dd * torch.where(a <= 2 * dd, 0.25, torch.where(a <= 4 * dd, 0.5, 1.0)), a - 6 * dd)
    assert ((val - act).abs() <= half * (1 + 2.0 ** -20) + slack)[live].all()
    assert (q[~live] == 0).all() and (s.view(torch.uint8)[~live] == 0).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,e,k,n,swiglu", [
    (8, 32, 7168, 4096, True), (8, 32, 2048, 7168, False),        # a token's eight experts
    (40, 4, 1024, 512, True), (40, 4, 1024, 512, False),          # up to 64 rows in all
    (768, 32, 4096, 2048, True), (768, 32, 1024, 4096, False),    # many experts, narrow tiles beside room for 128 rows
    (100, 1, 512, 256, True), (200, 2, 640, 384, False),          # few tiles
    (300, 3, 4096, 1024, True),
])
def test_few_rows(ops, fmt, m, e, k, n, swiglu):
    """The forms for few rows per expert, at the sizes where their tiles, stages and row slots differ."""
    gen = torch.Generator().manual_seed(m + e)
    cnt = torch.bincount(torch.randint(0, e, (m,), generator=gen), minlength=e).tolist()
    aq, as_ = random_fp4((m, k), fmt, gen)
    wq, ws = random_fp4((e, n, k), fmt, gen)
    ag, wg = (torch.full((1,), 0.002), torch.rand(e, generator=gen) * 0.02) if fmt == "nvfp4" else (None, None)
    off = offsets_of(cnt)
    if not swiglu:
        got = ops.grouped_gemm_fp4(*_dev(aq, as_, wq, ws, off, ag, wg))
        want, mag = _product64(values64(*_dev(aq, as_, ag)), values64(*_dev(wq, ws, wg)), off, m)
        assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * _acc_tol(k)).all()
        return
    # gate and up from the plain product; the SwiGLU form has to agree with it through its own definition
    gu = ops.grouped_gemm_fp4(*_dev(aq, as_, wq, ws, off, ag, wg)).double()
    q, s = ops.grouped_gemm_fp4_swiglu(*_dev(aq, as_, wq, ws, off, ag, wg))
    g, u = gu.chunk(2, -1)
    act = g * torch.sigmoid(g) * u
    # gu was rounded to bf16 (2^-8 relative in each factor, |silu'| <= 1.1 of the gate) on top of the 4-bit rounding: half a
    # step (a step is at most a third of the value, or half of the scale) and what is cut off above 6 scales (a sixteenth)
    val = values64(q, s)
    d = (s.double() if fmt == "nvfp4" else torch.exp2(s.view(torch.uint8).double() - 127)).repeat_interleave(16 if fmt == "nvfp4" else 32, -1)
    slack = 2.0 ** -8 * (1.1 * g.abs() * u.abs() + act.abs()) * 1.01 + act.abs() * 2.0 ** -12
    cut = torch.where(d <= 2.0 ** -8, act.abs(), act.abs() / 16)  # scales near the smallest e4m3 are rounded by up to half of themselves
    assert ((val - act).abs() <= torch.maximum(0.25 * d, act.abs() / 6) + cut + slack).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("split", ["1", "2", "4"])
@pytest.mark.parametrize("m,e,k,n,swiglu", [(40, 4, 1024, 512, True), (700, 3, 2176, 1024, False), (900, 2, 4352, 512, True)])
def test_tiles_shared_by_a_cluster(ops, fmt, split, m, e, k, n, swiglu, monkeypatch):
    monkeypatch.setenv("UMDK_CAM_EXPERT_NARROW", "1")
    monkeypatch.setenv("UMDK_CAM_EXPERT_SPLIT", split)
    test_few_rows(ops, fmt, m, e, k, n, swiglu)


def test_status_is_clean(ops):
    from umdk_original_b200.ops import cam_ops
    assert cam_ops.native_module().expert_ops_status()[0] == 0


def test_refusals(ops):
    from test_fp4_cpu import refusals
    for what, call in refusals(DEV):
        with pytest.raises(RuntimeError, match="umdk_cam_op_lib"):
            call()
    x = torch.randn(4, 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="device"):
        ops.quantize_fp4(x, 16, torch.ones(1))
    shifted = torch.empty(4 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(4, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.quantize_fp4(shifted, 16)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_offset_scale_arrays(ops, fmt):
    """Scales that start on a 4-byte but not on a 16-byte boundary, in sizes whose rows would allow wide loads."""
    gen = torch.Generator().manual_seed(8)
    aq, as_ = random_fp4((40, 512), fmt, gen)
    wq, ws = random_fp4((2, 256, 512), fmt, gen)
    off = offsets_of([17, 23])
    want = ops.grouped_gemm_fp4(*_dev(aq, as_, wq, ws, off))

    def moved(t):
        b = torch.zeros(t.numel() + 4, dtype=torch.uint8, device=DEV)
        b[4:] = t.view(torch.uint8).flatten().to(DEV)
        return b[4:].view(t.dtype).view(t.shape)
    assert torch.equal(ops.grouped_gemm_fp4(aq.to(DEV), moved(as_), wq.to(DEV), moved(ws), off.to(DEV)), want)


def test_graph_and_streams(ops):
    """Captured and replayed with new rows and new offsets; on a side stream; two calls in flight."""
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(96, 256, generator=gen).to(DEV, torch.bfloat16)
    w1 = ops.quantize_fp4((torch.randn(3, 512, 256, generator=gen) * 0.06).to(DEV), 16)
    w2 = ops.quantize_fp4((torch.randn(3, 256, 256, generator=gen) * 0.06).to(DEV), 16)
    off = offsets_of([32, 32, 32], device=DEV)

    def layer(x, off):
        q, s = ops.quantize_fp4(x, 16)
        q, s = ops.grouped_gemm_fp4_swiglu(q, s, *w1, off)
        return ops.grouped_gemm_fp4(q, s, *w2, off)

    first = layer(x, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = layer(x, off)
    b = layer(x, off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, first) and torch.equal(b, first)
    xs, offs = x.clone(), off.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(xs, offs)
    x2 = torch.randn(96, 256, generator=gen).to(DEV, torch.bfloat16)
    off2 = offsets_of([1, 60, 20], device=DEV)
    xs.copy_(x2)
    offs.copy_(off2)
    g.replay()
    assert torch.equal(y, layer(x2, off2))


def test_offsets_past_32_bits(ops):
    """Weights of more than 2^31 bytes of codes: the last expert's; rows behind 2^31 values."""
    e, n, k = 70, 8192, 8192
    gen = torch.Generator().manual_seed(11)
    wq = torch.zeros(e, n, k // 2, dtype=torch.uint8, device=DEV)
    ws = torch.zeros(e, n, k // 16, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    assert wq.numel() > 2 ** 31
    q, s = random_fp4((n, k), "nvfp4", gen, DEV)
    wq[-1] = q
    ws.view(torch.uint8)[-1] = s.view(torch.uint8)
    aq, as_ = random_fp4((33, k), "nvfp4", gen, DEV)
    off = torch.tensor([0] * e + [33], dtype=torch.int32, device=DEV)
    want, mag = _product64(values64(aq, as_), values64(q, s)[None], torch.tensor([0, 33]), 33)
    got = ops.grouped_gemm_fp4(aq, as_, wq, ws, off)
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * _acc_tol(k)).all()
    del wq, ws
    x = torch.zeros(2 ** 31 // 4096 + 3, 4096, dtype=torch.bfloat16, device=DEV)
    x[-2:] = torch.randn(2, 4096, generator=gen).to(DEV)
    q, s = ops.quantize_fp4(x, 32)
    wq2, ws2 = ops.quantize_fp4(x[-2:].contiguous(), 32)
    assert torch.equal(q[-2:], wq2) and torch.equal(s[-2:].view(torch.uint8), ws2.view(torch.uint8))
    assert (ops.dequantize_fp4(q, s)[-2:] != 0).any()


def test_wild_offsets_stay_inside(ops):
    from umdk_original_b200.ops import cam_ops
    gen = torch.Generator().manual_seed(12)
    aq, as_ = random_fp4((50, 256), "mxfp4", gen, DEV)
    wq, ws = random_fp4((3, 256, 256), "mxfp4", gen, DEV)
    for off in ([40, -7, 60, 10], [2 ** 31 - 1] * 4, [0, 0, 0, 10 ** 9]):
        o = torch.tensor(off, dtype=torch.int32, device=DEV)
        ops.grouped_gemm_fp4(aq, as_, wq, ws, o)
        ops.grouped_gemm_fp4_swiglu(aq, as_, wq, ws, o)
        torch.cuda.synchronize()
        assert cam_ops.native_module().expert_ops_status()[0] == 0
