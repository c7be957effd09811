"""quantize_fp4 at the ends of its range: the CUDA key against the CPU key, code by code, and against the definition."""
import pytest
import torch

from fp4_cases import quantise64, values64

pytestmark = pytest.mark.gpu

DEV = "cuda"
POINTS = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])  # every half-way point, and the top
ROUNDED = torch.tensor([0, 1, 1, 2, 2, 4, 4, 6.0], dtype=torch.float64)


@pytest.fixture(scope="module")
def ops():
    from umdk_original_b200 import ops
    return ops


def codes(q):
    """e2m1 values of packed codes, without scales."""
    return values64(q.cpu(), torch.ones(*q.shape[:-1], 1).to(torch.float8_e4m3fn))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("exponent", [-60, -61, -100, -120, -128, -130])
def test_tiny_global_scale(ops, dtype, exponent):
    """Scale times global scale down to 2^-142, where 1 / d is no fp32 number; values and scales are exact."""
    g = torch.tensor([2.0 ** exponent], dtype=torch.float64).float()
    for scale in (1.0, 1.625, 2.0 ** -9):
        x = (torch.cat([POINTS, -POINTS]).double() * scale * g.double()).reshape(1, 16).to(dtype)
        if dtype == torch.bfloat16 and not torch.equal(x.double(), torch.cat([POINTS, -POINTS])[None].double() * scale * g.double()):
            continue  # bf16 subnormals hold fewer bits
        q, s = ops.quantize_fp4(x.to(DEV), 16, g.to(DEV))
        assert float(s.cpu().double()) == scale
        assert torch.equal(codes(q)[0], torch.cat([ROUNDED, -ROUNDED]))
        cq, cs = ops.quantize_fp4(x, 16, g)
        assert torch.equal(q.cpu(), cq) and torch.equal(s.cpu().view(torch.uint8), cs.view(torch.uint8))


def test_values_far_above_the_scale(ops):
    """A global scale far too small: the block scale is cut to 448, quotients overflow fp32 and saturate with their sign."""
    x = torch.tensor([3e38, -3e38, 1e30, -1e30, 1e-3, -1e-3, 0.0, 448e-6 * 2.5] * 2).reshape(1, 16)
    g = torch.tensor([1e-6])
    q, s = ops.quantize_fp4(x.to(DEV), 16, g.to(DEV))
    assert float(s.cpu().double()) == 448.0
    want, _ = quantise64(x, 16, g)
    # The divisor, scale x global scale, is rounded once to fp32: it moves the quotient by 2^-24 of itself at most, across a half-way
    # point only if it lies that near to one (the last value of each half does: 448e-6 x 2.5 in fp32)
    quotient = (x.double() / (448.0 * g.double())).abs()
    clear = ((quotient[..., None] / POINTS[:7].double() - 1).abs() > 2.0 ** -23).all(-1)
    assert int((~clear).sum()) == 2 and torch.equal(codes(q)[clear], want[clear])
    cq, cs = ops.quantize_fp4(x, 16, g)
    assert torch.equal(codes(q), codes(cq)) and torch.equal(s.cpu().view(torch.uint8), cs.view(torch.uint8))


@pytest.mark.parametrize("g", [None, 0.0123])
def test_finite_values_beside_an_infinity(ops, g):
    """They are divided like all others: quotients half-way between two codes go to the even one."""
    gs = None if g is None else torch.tensor([g])
    d = 448.0 * (1.0 if g is None else float(gs))
    x = torch.cat([POINTS, -POINTS]) * torch.tensor(d)
    x[7], x[15] = float("inf"), float("-inf")
    q, s = ops.quantize_fp4(x.reshape(1, 16).to(DEV), 16, None if gs is None else gs.to(DEV))
    cq, cs = ops.quantize_fp4(x.reshape(1, 16), 16, gs)
    assert torch.equal(codes(q), codes(cq)) and torch.equal(s.cpu().view(torch.uint8), cs.view(torch.uint8))
    if g is None:
        assert torch.equal(codes(q)[0], torch.cat([ROUNDED, -ROUNDED]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,g", [(16, None), (16, 0.0123), (16, 1e-30), (16, 3e-39), (16, 1e30), (16, 2e38), (32, None)])
def test_same_codes_as_the_cpu_key(ops, dtype, block, g):
    """Rows whose magnitudes span the type's whole range, block by block."""
    gen = torch.Generator().manual_seed(21)
    top = 38.0 if dtype != torch.float16 else 4.0
    x = torch.randn(64, 40 * block, generator=gen)
    low = {torch.float32: -44.0, torch.bfloat16: -40.0, torch.float16: -7.0}[dtype]
    x *= 10.0 ** (torch.rand(64, 40, generator=gen, dtype=torch.float64) * (top - low - 1) + low).float().repeat_interleave(block, 1)
    x = x.to(dtype)
    gs = None if g is None else torch.tensor([g], dtype=torch.float64).float()
    q, s = ops.quantize_fp4(x.to(DEV), block, None if gs is None else gs.to(DEV))
    cq, cs = ops.quantize_fp4(x, block, gs)
    assert torch.equal(s.cpu().view(torch.uint8), cs.view(torch.uint8))
    assert torch.equal(codes(q), codes(cq))


def test_infinite_divisor(ops):
    """448 x global scale past fp32 beside an infinity: finite values are nothing in that scale."""
    x = torch.cat([torch.full((1, 15), -3e38), torch.full((1, 1), float("inf"))], -1)
    g = torch.tensor([1e37])
    q, s = ops.quantize_fp4(x.to(DEV), 16, g.to(DEV))
    cq, cs = ops.quantize_fp4(x, 16, g)
    assert torch.equal(s.cpu().view(torch.uint8), cs.view(torch.uint8))
    assert (codes(q)[0, :15] == 0).all() and (codes(cq)[0, :15] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,g", [(16, None), (16, 0.0123), (16, 1e-20), (32, None)])
def test_bytes_and_the_sign_of_zero(ops, dtype, block, g):
    """Packed bytes are the CPU key's, zeros of both signs and negative values that round to zero among them."""
    gen = torch.Generator().manual_seed(22)
    x = torch.randn(16, 8 * block, generator=gen)
    x[:, ::5] = -0.0
    x[:, 1::5] = 0.0
    x[:, 2::7] *= -1e-4
    x[3], x[4] = 0.0, -0.0
    x[5, :block] = -1e-7  # with some scales these blocks get the scale zero
    x = x.to(dtype)
    gs = None if g is None else torch.tensor([g])
    q, s = ops.quantize_fp4(x.to(DEV), block, None if gs is None else gs.to(DEV))
    cq, cs = ops.quantize_fp4(x, block, gs)
    assert torch.equal(s.cpu().view(torch.uint8), cs.view(torch.uint8))
    assert torch.equal(q.cpu(), cq)
    nibbles = torch.stack([cq & 15, cq >> 4], -1).flatten(-2)
    assert torch.equal(nibbles >> 3, torch.signbit(x).to(torch.uint8))
