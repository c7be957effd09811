"""Global scales of an nvfp4 expert MLP from sample rows."""
import pytest
import torch

from fp4_cases import offsets_of
from umdk_original_b200 import ops
from umdk_original_b200.models import ExpertMLP


def build(device):
    m = ExpertMLP(2, 128, 128, device=device, seed=3)
    x = torch.randn(15, 128, generator=torch.Generator().manual_seed(4)).to(device, torch.bfloat16)
    return m, x, offsets_of([5, 4], head=2, device=device)


def errors(device, size):
    m, x, off = build(device)
    x = x * size
    x[:2], x[11:] = float("nan"), float("inf")  # rows of no expert
    layer = m.quantized("nvfp4").calibrate(x, off)
    q, s = ops.quantize_fp4(x, 16, layer.x_gs)
    rows, back = x[2:11].float(), ops.dequantize_fp4(q, s, layer.x_gs, torch.float32)[2:11]
    with torch.no_grad():
        want, got = m(x, off)[2:11].float(), layer(x, off)[2:11].float()
    return (back - rows).norm() / rows.norm(), (got - want).norm() / want.norm()


def check(device, size):
    """A value is off by a quarter of the scale d or a sixth of itself at most, or by a sixteenth more where the rounded scale cuts it;
    d is a sixth of the block's largest value, give or take a sixteenth: sqrt(1.13 / 36 + 1 / 36) + 1 / 16 of a block's norm at most.
    Gaussian values are off by a tenth of their norm, independently of each other, so four such operands and the products
    between them (gate and up, each off by 0.14) leave about a quarter."""
    rows, result = errors(device, size)
    assert rows < 0.31 and result < 0.35


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 1e4])
def test_rows_of_any_size(size):
    check("cpu", size)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 1e4])
def test_rows_of_any_size_on_the_gpu(size):
    check("cuda", size)


def test_what_calibration_refuses_and_leaves():
    m, x, off = build("cpu")
    bad = x.clone()
    bad[4, 7] = float("nan")
    with pytest.raises(ValueError, match="rows hold NaN"):
        m.quantized("nvfp4").calibrate(bad, off)
    zero = m.quantized("nvfp4").calibrate(torch.zeros_like(x), off)
    assert float(zero.x_gs) == 1.0 and float(zero.act_gs) == 1.0
    none = m.quantized("nvfp4").calibrate(x, offsets_of([0, 0]))
    assert float(none.x_gs) == 1.0
    mx = m.quantized("mxfp4").calibrate(x, off)
    assert mx.x_gs is None and mx.act_gs is None
