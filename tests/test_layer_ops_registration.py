"""What PyTorch's own checker says of the operators round the experts; compiled programs; forward mode and functorch."""
import pytest
import torch
from torch.library import opcheck

from umdk_original_b200 import ops
from umdk_original_b200.ops import cam_ops

pytestmark = pytest.mark.skipif(not cam_ops.native_loaded(), reason="native extension not built")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# the schema test sums its inputs, which PyTorch does not do for 8-bit floats
NO_SCHEMA = ("test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
ALL = ("test_schema", *NO_SCHEMA)
# the last one adds all outputs up in place, beginning with the first: not where that holds integers; test_compiled_program stands in
INTEGERS_FIRST = ALL[:-1]


def cases(dev):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    x, res, w = r(6, 128).bfloat16(), r(6, 128), r(128).bfloat16()
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    lib = torch.ops.umdk_cam_op_lib
    yield lib.rms_norm, (x, w), ALL
    yield lib.rms_norm, (leaf(x), leaf(w)), ALL
    yield lib.add_rms_norm, (x, res, w), ALL
    yield lib.add_rms_norm, (leaf(x), leaf(res), leaf(w)), ALL
    yield lib.add_rms_norm, (leaf(x), leaf(x), w), ALL
    yield lib.rms_norm_train, (x, None, w), ALL
    _, s, rstd = ops.rms_norm_train(x, res, w)
    yield lib.rms_norm_train, (x, res, w), ALL
    yield lib.rms_norm_backward, (x, s, s, w, rstd), ALL
    yield lib.rms_norm_backward, (x, None, x, w, rstd, True, False, False), ALL
    for mode in (2, 3, 4):
        yield lib.rms_norm_quant, (x, w, mode), NO_SCHEMA
        yield lib.rms_norm_quant, (x, w, mode, res, 1e-6, True), NO_SCHEMA
    logits, bias = r(6, 8), r(8)
    yield lib.moe_route, (logits, 2), ALL
    yield lib.moe_route, (leaf(logits), 2, bias, "sigmoid", 4, 2, 2, False, 2.0), INTEGERS_FIRST
    idx, wt = ops.moe_route(logits, 2)
    yield lib.moe_route_backward, (wt, logits, idx), ALL
    yield lib.moe_group_rows, (x, idx, 8), ALL
    yield lib.moe_group_rows, (x, idx, 8, r(6, 3)), ALL
    yield lib.moe_group_rows, (leaf(x), idx, 8), ALL
    rows, _, _, slots = ops.moe_group_rows(x, idx, 8)
    yield lib.moe_ungroup_rows, (rows, slots), ALL
    yield lib.moe_ungroup_rows, (leaf(rows), slots, leaf(wt), leaf(x)), ALL
    yield lib.moe_ungroup_rows, (rows, slots, leaf(wt)), ALL
    yield lib.moe_ungroup_rows_backward, (x, rows, slots, wt), ALL
    yield lib.moe_ungroup_rows_backward, (x, rows, slots, None, True, False), ALL


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("i", range(26))
def test_opcheck(device, i):
    op, args, tests = list(cases(device))[i]
    opcheck(op.default, args, test_utils=tests)


def test_all_cases_are_checked():
    assert len(list(cases("cpu"))) == 26


@pytest.mark.parametrize("device", DEVICES)
def test_opcheck_of_rows_that_are_only_numbered(device):
    gen = torch.Generator().manual_seed(2)
    dout, wt = torch.randn(3, 64, generator=gen).to(device), torch.rand(3, 2, generator=gen).to(device)
    slots = torch.tensor([[0, 4], [-1, 2], [5, 1]], dtype=torch.int32, device=device)
    lib = torch.ops.umdk_cam_op_lib
    opcheck(lib.moe_ungroup_rows_backward.default, (dout, dout.new_empty(6, 0), slots, wt, True, False), test_utils=ALL)
    opcheck(lib.moe_ungroup_rows.default, (torch.randn(6, 64, generator=gen).to(device).requires_grad_(), slots, wt), test_utils=ALL)


@pytest.mark.parametrize("device", DEVICES)
def test_compiled_program(device):
    """A traced program of all of them, with its backward pass, gives the bits of the eager one."""
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen).to(device)  # noqa: E731
    x, res, w, gate = r(10, 64).bfloat16(), r(10, 64).bfloat16(), r(64).bfloat16(), r(8, 64).bfloat16()
    dy, ds = r(10, 64).bfloat16(), r(10, 64).bfloat16()

    def program(x, res, w, gate):
        y, s = ops.add_rms_norm(x, res, w)
        idx, wt = ops.moe_route(y @ gate.t(), 3, None, "softmax", 4, 2)
        rows, _, _, slots = ops.moe_group_rows(y, idx, 8)
        return ops.moe_ungroup_rows(rows * 2, slots, wt, s), s
    got = []
    for fn in (program, torch.compile(program, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in (x, res, w, gate)]
        out = fn(*leaves)
        got.append([t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (dy, ds))))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(no_grad):
    import torch.autograd.forward_ad as fwad
    x, w, idx = torch.randn(6, 64), torch.randn(64), torch.zeros(6, 1, dtype=torch.int64)
    slots = torch.arange(6, dtype=torch.int32)[:, None].contiguous()
    calls = [lambda t: ops.rms_norm(t, w), lambda t: ops.rms_norm(x, t[0]), lambda t: ops.add_rms_norm(x, t, w), lambda t: ops.moe_route(t, 2),
             lambda t: ops.moe_group_rows(t, idx, 2), lambda t: ops.moe_ungroup_rows(t, slots), lambda t: ops.moe_ungroup_rows(x, slots, None, t),
             lambda t: ops.moe_ungroup_rows(x, slots, t[:, :1].contiguous())]
    for call in calls:
        with torch.set_grad_enabled(not no_grad), fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(fwad.make_dual(x, torch.ones_like(x)))


def test_functorch():
    """Batches of calls are computed one by one; gradients inside torch.func are refused, not left out."""
    x, w = torch.randn(3, 6, 64), torch.randn(64)
    got = torch.func.vmap(lambda t: ops.rms_norm(t, w))(x)
    assert torch.equal(got, torch.stack([ops.rms_norm(t, w) for t in x]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ops.rms_norm(x[0], t).sum())(w)
