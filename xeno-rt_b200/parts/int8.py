"""Products of 8-bit integers: matrices and rows of activations held as int8 with one 32-bit scale a row.

A product of x and W is sum_k x[m, k] W[n, k] = scale_x[m] * scale_w[n] * sum_k of their integers, whose sum is exact.  W is
laid out once, when the model is built; x is rounded on the way into every product: by the norm or the gate that makes it
where those can (``RMSNorm.forward_int8``, ``SwiGLUFeedForward``), else by a kernel of its own."""
from __future__ import annotations

import torch

from ..core import KernelError
from ..csrc import ops


class Int8Matrix:
    """A weight [out, in] as ``codes`` int8 and ``scales`` float32 [out].  ``constant``: no kernel that may still run wrote the
    codes; products of few rows then read them while the kernel before finishes."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, constant: bool = False):
        self.codes, self.scales, self.constant = codes, scales, constant

    @classmethod
    def of(cls, weight: torch.Tensor) -> "Int8Matrix":
        """The nearest codes of a float32 or bfloat16 weight, a scale a row.  Waits until they are written (they are constant from
        here on), so not inside a stream capture."""
        if weight.is_cuda and torch.cuda.is_current_stream_capturing():
            raise KernelError("a matrix is laid out in 8 bits outside of stream captures")
        codes = ops.int8_rows(weight.shape[0], weight.shape[1], weight.device)
        scales = torch.empty(weight.shape[0], dtype=torch.float32, device=weight.device)
        ops.quantize_rows(codes, scales, weight.contiguous())
        torch.cuda.current_stream(weight.device).synchronize()
        return cls(codes, scales, constant=True)

    @property
    def shape(self):
        return self.codes.shape

    def __getitem__(self, rows: slice) -> "Int8Matrix":
        return Int8Matrix(self.codes[rows], self.scales[rows], self.constant)


class Int8Rows:
    """Rows of activations [T, width] as ``codes`` int8 and ``scales`` float32 [T]."""

    def __init__(self, rows: int, width: int, device):
        self.codes = ops.int8_rows(rows, width, device)
        self.scales = torch.empty(rows, dtype=torch.float32, device=device)

    @classmethod
    def of(cls, x: torch.Tensor) -> "Int8Rows":
        rows = cls(x.shape[0], x.shape[1], x.device)
        ops.quantize_rows(rows.codes, rows.scales, x)
        return rows

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def dtype(self):
        return self.codes.dtype


def product(out: torch.Tensor, x, weight: Int8Matrix, accumulate: bool) -> None:
    """out = x . weight^T, or added into a float32 ``out``; x ``Int8Rows``, or a tensor that is rounded to that first."""
    if not isinstance(x, Int8Rows):
        x = Int8Rows.of(x)
    ops.gemm_int8(out, x.codes, x.scales, weight.codes, weight.scales, accumulate=accumulate, constant_weight=weight.constant)
