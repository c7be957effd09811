"""Ops of ``torch.ops.umdk_cam_op_lib`` (same six names as the reference) and the CPU oracle."""
from . import reference  # noqa: F401
from .cam_ops import native_loaded, native_module, ops  # noqa: F401

fused_deep_moe = ops.fused_deep_moe
get_dispatch_layout = ops.get_dispatch_layout
moe_dispatch_prefill = ops.moe_dispatch_prefill
moe_combine_prefill = ops.moe_combine_prefill
moe_dispatch_shmem = ops.moe_dispatch_shmem
moe_combine_shmem = ops.moe_combine_shmem
moe_dispatch_prefill_quant = ops.moe_dispatch_prefill_quant
grouped_gemm_fp8 = ops.grouped_gemm_fp8
grouped_gemm_fp8_swiglu = ops.grouped_gemm_fp8_swiglu

# The operators that need no Buffer are looked up when they are first used: the package, and with it the build, can be
# imported beside an extension that was built before they existed.  They have one overload each, which is called directly: the
# choice among overloads costs 0.6 us of the 7 that such a call takes on the host.
_EXPERT_OPS = ("quantize_fp4", "dequantize_fp4", "grouped_gemm_fp4", "grouped_gemm_fp4_swiglu", "grouped_mlp",
               "grouped_mlp_train", "grouped_mlp_backward", "rms_norm", "add_rms_norm", "rms_norm_train", "rms_norm_backward",
               "rms_norm_quant", "moe_route", "moe_route_backward", "moe_group_rows", "moe_ungroup_rows", "moe_ungroup_rows_backward")


def check_expert_ops(device=None) -> None:
    """Waits for the device (default: the current one) and raises ``CamError`` if a wait inside a product of the operators above ran
    out there since the last check (results since then mean nothing), the counterpart of ``Buffer.check``.  Without a check the next
    product on that device is refused, and all further ones, until this has reported and cleared it."""
    import torch

    from ..utils.errors import raise_for_status
    if not torch.cuda.is_available():
        return
    with torch.cuda.device(device):
        code, who, block, detail = native_module().expert_ops_status(True)
    raise_for_status(code, who, detail, block)


def __getattr__(name):
    if name not in _EXPERT_OPS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    globals()[name] = op = getattr(ops, name).default
    return op
