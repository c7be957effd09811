"""A wait that runs out inside an expert product is reported.  The kernels' record is written by the host here: no wait is made to fail."""
import pytest
import torch

from fp4_cases import offsets_of, random_fp4
from umdk_original_b200 import ops
from umdk_original_b200.ops import cam_ops
from umdk_original_b200.utils.errors import CamError, MoeCommTimeout


def test_check_raises_what_the_record_says(monkeypatch):
    class Native:
        record = (5, 1, 17, 3)  # code, who, block, detail

        def expert_ops_status(self, clear):
            assert clear
            got, self.record = self.record, (0, 0, 0, 0)
            return got
    native = Native()
    monkeypatch.setattr(ops, "native_module", lambda: native)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "device", lambda d: torch.no_grad())
    with pytest.raises(MoeCommTimeout) as err:
        ops.check_expert_ops()
    assert (err.value.code, err.value.who, err.value.detail, err.value.block) == (5, 1, 3, 17)
    ops.check_expert_ops()


def test_check_without_a_gpu():
    if not torch.cuda.is_available():
        ops.check_expert_ops()


@pytest.mark.gpu
def test_products_are_refused_until_the_check():
    dev = torch.device("cuda", 0)
    native = cam_ops.native_module()
    gen = torch.Generator().manual_seed(1)
    aq, as_ = random_fp4((40, 256), "nvfp4", gen, dev)
    wq, ws = random_fp4((2, 256, 256), "nvfp4", gen, dev)
    off = offsets_of([17, 23], device=dev)
    x = torch.randn(40, 64, generator=gen).to(dev, torch.bfloat16)
    w1 = torch.randn(2, 64, 64, generator=gen).to(dev, torch.bfloat16).requires_grad_()
    w2 = torch.randn(2, 64, 32, generator=gen).to(dev, torch.bfloat16)
    calls = [lambda: ops.grouped_gemm_fp4(aq, as_, wq, ws, off), lambda: ops.grouped_gemm_fp4_swiglu(aq, as_, wq, ws, off)[0],
             lambda: ops.grouped_mlp(x, w1, w2, off).detach(), lambda: ops.grouped_mlp(x[:1], w1, w2, off).detach()]
    want = [c() for c in calls]
    y = ops.grouped_mlp(x, w1, w2, off)
    ops.check_expert_ops()
    native.expert_ops_set_status(5, 1, 3, 17)
    for call in calls + [lambda: torch.autograd.grad(y, w1, torch.ones_like(y))]:
        with pytest.raises(RuntimeError, match="gave up.*mbarrier.*check_expert_ops"):
            call()
    assert native.expert_ops_status() == (5, 1, 17, 3) == native.expert_ops_status()  # looking does not clear
    with pytest.raises(CamError, match="code=5, who=1, detail=3, block=17"):
        ops.check_expert_ops(dev)
    ops.check_expert_ops()
    assert all(torch.equal(c(), t) for c, t in zip(calls, want))


@pytest.mark.gpu
def test_first_product_of_a_process_may_be_captured():
    """The status word is allocated by the first product, which a capture must not make fail."""
    import subprocess
    import sys
    from pathlib import Path
    prog = """
import torch
from umdk_original_b200 import ops
x = torch.randn(300, 64, device="cuda").bfloat16()
w1, w2 = torch.randn(2, 512, 64, device="cuda").bfloat16(), torch.randn(2, 64, 256, device="cuda").bfloat16()
off = torch.tensor([0, 140, 300], dtype=torch.int32, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.grouped_mlp(x, w1, w2, off)
g.replay()
ops.check_expert_ops()
assert torch.equal(y, ops.grouped_mlp(x, w1, w2, off)) and y.abs().sum() > 0
"""
    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", prog], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
