"""What PyTorch's own checker says of the expert operators: schemas, shapes of traced tensors, autograd registration, compiled programs
with static and dynamic sizes."""
import pytest
import torch
from torch.library import opcheck

from fp4_cases import offsets_of, random_fp4
from umdk_original_b200 import ops
from umdk_original_b200.ops import cam_ops

pytestmark = pytest.mark.skipif(not cam_ops.native_loaded(), reason="native extension not built")
# the schema test sums its inputs, which PyTorch does not do for 8-bit floats
NO_SCHEMA = ("test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
ALL = ("test_schema", *NO_SCHEMA)


def cases(dev):
    gen = torch.Generator().manual_seed(0)
    x, w1, w2 = (torch.randn(*s, generator=gen).to(dev, torch.bfloat16) / 4 for s in ((13, 64), (3, 32, 64), (3, 64, 16)))
    off = offsets_of([3, 0, 4], 1, dev)
    lib = torch.ops.umdk_cam_op_lib
    _, act, gu = ops.grouped_mlp_train(x, w1, w2, off)
    act, gu = act.nan_to_num(), gu.nan_to_num()  # rows of no expert hold nothing defined
    act[:1], act[8:], gu[:1], gu[8:] = 0, 0, 0, 0
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    yield lib.grouped_mlp, (x, w1, w2, off), ALL
    yield lib.grouped_mlp, (*leaves, off), ALL
    yield lib.grouped_mlp, (x, leaves[1], w2, off), ALL
    yield lib.grouped_mlp_backward, (x, x, w1, w2, off, act, gu), ALL
    yield lib.grouped_mlp_backward, (x, x, w1, w2, off, act, gu, False, True, False), ALL
    yield lib.grouped_mlp_keep, (x,), ALL
    for fmt, block in (("nvfp4", 16), ("mxfp4", 32)):
        yield lib.quantize_fp4, (x, block), ALL
        aq, as_ = random_fp4((10, 128), fmt, gen, dev)
        wq, ws = random_fp4((3, 256, 128), fmt, gen, dev)
        yield lib.dequantize_fp4, (aq, as_), NO_SCHEMA
        yield lib.dequantize_fp4, (aq, as_, None, torch.float32), NO_SCHEMA
        yield lib.grouped_gemm_fp4, (aq, as_, wq, ws, off), NO_SCHEMA
        yield lib.grouped_gemm_fp4_swiglu, (aq, as_, wq, ws, off), NO_SCHEMA


@pytest.mark.parametrize("i", range(16))
def test_opcheck(i):
    op, args, tests = list(cases("cpu"))[i]
    opcheck(op.default, args, test_utils=tests)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(16))
def test_opcheck_on_the_gpu(i):
    op, args, tests = list(cases("cuda"))[i]
    opcheck(op.default, args, test_utils=tests)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_compiled_4_bit_layer(device, fmt):
    from umdk_original_b200.models import ExpertMLP
    layer = ExpertMLP(2, 128, 128, device=device, seed=3).quantized(fmt)
    fn = torch.compile(lambda x, off: layer(x, off) * 2, backend="aot_eager", fullgraph=True)
    gen = torch.Generator().manual_seed(4)
    for cnt in ([5, 4], [0, 30]):
        x, off = torch.randn(sum(cnt) + 3, 128, generator=gen).to(device, torch.bfloat16), offsets_of(cnt, 1, device)
        assert torch.equal(fn(x, off), layer(x, off) * 2)
