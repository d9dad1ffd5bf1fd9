"""y = x . W^T for a weight stored [out, in] as the reference stores every matrix
(crates/xrt-models/src/llama.rs:447-486, no bias anywhere).  Chooses the kernel by dtype and size."""
from __future__ import annotations

import torch

from ..core import KernelError
from ..csrc import ops
from .int8 import Int8Matrix
from .int8 import product as int8_product


def linear(x, weight: torch.Tensor, out_dtype=None, accumulate_into: torch.Tensor | None = None, then_norm=None,
           out: torch.Tensor | None = None):
    """Returns x . weight^T in ``out_dtype`` (default float32), or, with ``accumulate_into`` (a
    float32 tensor [M, N], the residual stream), adds the product into it in place and returns it.
    Accumulation is 32-bit in every kernel.  ``x`` may be a ``PendingNorm`` (see parts/norm.py).
    ``then_norm`` (an RMSNorm part, with ``accumulate_into``): if the kernel that runs can prepare that
    norm of the new residual on its way, the result is (residual, PendingNorm), else (residual, None).
    ``out`` (a contiguous tensor [M, N]): the product is written there instead of into a new tensor.
    ``weight`` may be an ``Int8Matrix`` and ``x`` then ``Int8Rows`` too (see parts/int8.py)."""
    if out is not None and (accumulate_into is not None or tuple(out.shape) != (x.shape[0], weight.shape[0])
                            or not out.is_contiguous()):
        raise KernelError("linear: out must be a contiguous [rows, weight rows] tensor, and not given with accumulate_into")
    from .norm import PendingNorm
    if isinstance(x, PendingNorm):
        from . import linear_bf16
        if out is None:
            out = torch.empty((x.shape[0], weight.shape[0]), dtype=out_dtype or torch.float32, device=x.device)
        linear_bf16.run_pending(out, x, weight)
        return out
    m = x.shape[0]
    n = weight.shape[0]
    if accumulate_into is not None:
        out = accumulate_into
        if out.dtype != torch.float32:
            raise KernelError("linear: the residual stream must be float32")
    elif out is None:
        out = torch.empty((m, n), dtype=out_dtype or torch.float32, device=x.device)
    accumulate = accumulate_into is not None
    pending = None
    if m > 0:
        done = False
        if isinstance(weight, Int8Matrix):
            int8_product(out, x, weight, accumulate)
            done = True
        elif weight.dtype == torch.bfloat16 and x.dtype == torch.bfloat16:
            from . import linear_bf16
            if accumulate and then_norm is not None:
                pending = linear_bf16.run_with_norm(out, x, weight, then_norm)
                done = pending is not None
            done = done or linear_bf16.run(out, x, weight, accumulate)
        if not done:
            ops.gemm_reference(out, x, weight, accumulate=accumulate)
    return (out, pending) if then_norm is not None else out
