"""4-bit operators on the CPU key: definitions in 64 bits, and what is refused."""
import pytest
import torch

from fp4_cases import offsets_of, quantise64, random_fp4, values64
from umdk_original_b200 import ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,g", [(16, None), (16, 0.25), (32, None)])
def test_quantise_and_back(dtype, block, g):
    x = (torch.randn(5, 96, generator=torch.Generator().manual_seed(1)) * 3).to(dtype)
    gs = None if g is None else torch.tensor([g])
    q, s = ops.quantize_fp4(x, block, gs)
    want_q, want_s = quantise64(x, block, gs)
    assert torch.equal(values64(q, torch.ones(5, 1).to(torch.float8_e4m3fn)), want_q)
    assert torch.equal(s.float().double(), want_s)
    v = ops.dequantize_fp4(q, s, gs, torch.float32)
    assert torch.equal(v.double(), values64(q, s, gs))  # g is a power of two: nothing rounds


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_products(fmt):
    gen = torch.Generator().manual_seed(2)
    off = offsets_of([3, 0, 4], head=1)
    aq, as_ = random_fp4((10, 128), fmt, gen)
    wq, ws = random_fp4((3, 256, 128), fmt, gen)
    y = ops.grouped_gemm_fp4(aq, as_, wq, ws, off)
    a, w = values64(aq, as_), values64(wq, ws)
    for lo, hi, e in ((1, 4, 0), (4, 8, 2)):
        want, mag = a[lo:hi] @ w[e].T, a[lo:hi].abs() @ w[e].abs().T
        # fp32 sums of 128 exact products, one rounding to bf16
        assert ((y[lo:hi].double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * 128 * 2.0 ** -24).all()
    assert (y[0] == 0).all() and (y[8:] == 0).all()
    q, s = ops.grouped_gemm_fp4_swiglu(aq, as_, wq, ws, off)
    assert q.shape == (10, 64) and s.shape == (10, 128 // (16 if fmt == "nvfp4" else 32))


def test_meta_shapes():
    for fmt in ("nvfp4", "mxfp4"):
        gen = torch.Generator().manual_seed(2)
        aq, as_ = random_fp4((10, 128), fmt, gen, "meta")
        wq, ws = random_fp4((3, 256, 128), fmt, gen, "meta")
        off = offsets_of([3, 0, 4], device="meta")
        assert ops.grouped_gemm_fp4(aq, as_, wq, ws, off).shape == (10, 256)
        q, s = ops.grouped_gemm_fp4_swiglu(aq, as_, wq, ws, off)
        assert q.shape == (10, 64) and s.shape == (10, 128 // (16 if fmt == "nvfp4" else 32)) and s.dtype == as_.dtype
    q, s = ops.quantize_fp4(torch.empty(4, 64, device="meta", dtype=torch.bfloat16), 32)
    assert q.shape == (4, 32) and s.shape == (4, 2) and ops.dequantize_fp4(q, s).shape == (4, 64)


def refusals(device):
    """(what is wrong, call) of every refusal that needs no second device."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(4, 64).to(torch.bfloat16).to(device)
    one, two = torch.ones(1, device=device), torch.ones(2, device=device)
    off = offsets_of([2, 2], device=device)
    aq, as_ = random_fp4((4, 128), "nvfp4", gen, device)
    wq, ws = random_fp4((2, 256, 128), "nvfp4", gen, device)
    maq, mas = random_fp4((4, 128), "mxfp4", gen, device)
    mwq, mws = random_fp4((2, 256, 128), "mxfp4", gen, device)
    oq, os_ = random_fp4((4, 96), "nvfp4", gen, device)
    owq, ows = random_fp4((2, 256, 96), "nvfp4", gen, device)
    nwq, nws = random_fp4((2, 144, 128), "nvfp4", gen, device)
    hwq, hws = random_fp4((2, 128, 128), "nvfp4", gen, device)
    g, sw = ops.grouped_gemm_fp4, ops.grouped_gemm_fp4_swiglu
    return [
        ("block", lambda: ops.quantize_fp4(x, 64)),
        ("last dimension", lambda: ops.quantize_fp4(x[:, :24].contiguous(), 16)),
        ("last dimension", lambda: ops.quantize_fp4(x[:, :48].contiguous(), 32)),
        ("contiguous", lambda: ops.quantize_fp4(x.t(), 16)),
        ("type", lambda: ops.quantize_fp4(x.to(torch.int32), 16)),
        ("mx global scale", lambda: ops.quantize_fp4(x, 32, one)),
        ("two global scales for rows", lambda: ops.quantize_fp4(x, 16, two)),
        ("global scale type", lambda: ops.quantize_fp4(x, 16, one.double())),
        ("scale type", lambda: ops.dequantize_fp4(aq, as_.float())),
        ("scale shape", lambda: ops.dequantize_fp4(aq, as_[:, :4].contiguous())),
        ("output type", lambda: ops.dequantize_fp4(aq, as_, None, torch.float64)),
        ("formats differ", lambda: g(aq, as_, mwq, mws, off)),
        ("K", lambda: g(oq, os_, owq, ows, off)),
        ("K of the operands", lambda: g(oq, os_, wq, ws, off)),
        ("N", lambda: g(aq, as_, nwq, nws, off)),
        ("2I", lambda: sw(aq, as_, hwq, hws, off)),
        ("offsets", lambda: g(aq, as_, wq, ws, off[:-1].contiguous())),
        ("offsets type", lambda: g(aq, as_, wq, ws, off.long())),
        ("mx global scale of the rows", lambda: g(maq, mas, mwq, mws, off, one)),
        ("weights' global scales", lambda: g(aq, as_, wq, ws, off, one, one)),
        ("strided rows", lambda: g(aq[::2], as_[::2], wq, ws, off)),
    ]


@pytest.mark.parametrize("i", range(21))
def test_refusals(i):
    what, call = refusals("cpu")[i]
    with pytest.raises(RuntimeError, match="umdk_cam_op_lib"):
        call()
