"""Every quotient of two bfloat16 numbers that a row's code can be: the codes are those of IEEE's 32-bit division."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("exponent", [-118, -60, 0, 1, 60, 126])
@pytest.mark.parametrize("width", [1280, 4100])
def test_every_pair_of_16_bit_numbers(exponent, width):
    """A row for each of the 128 significands of its largest value, and in it every number down to 2^-9 of that (whose code is 0).
    The scale is the 32-bit quotient of the largest by 127, the code the whole number nearest to the 32-bit quotient by the scale."""
    from xeno_rt_b200.csrc import ops
    significands = 1 + np.arange(128, dtype=np.float64) / 128
    largest = significands * 2.0 ** exponent
    numbers = (significands[None, :] * 2.0 ** (exponent - np.arange(10, dtype=np.float64)[:, None])).reshape(-1)
    x = np.zeros((128, width))
    x[:, :1280] = np.where(numbers[None, :] <= largest[:, None], numbers[None, :], 0.0)
    x[:, 1::2] *= -1
    x[:, 0] = largest
    x = x.astype(np.float32)
    codes, scales = ops.int8_rows(128, width, DEV), torch.empty(128, device=DEV)
    rows = torch.from_numpy(x).to(DEV).bfloat16()
    x = rows.float().cpu().numpy()  # (numbers below 2^-126 have fewer bits)
    ops.quantize_rows(codes, scales, rows)
    scale = np.maximum(np.abs(x).max(axis=1) / np.float32(127), np.float32(2.0 ** -126))
    assert scale.dtype == np.float32 and np.array_equal(scales.cpu().numpy(), scale)
    assert np.array_equal(codes.cpu().numpy(), np.rint(x / scale[:, None]))


@pytest.mark.parametrize("rows", [64, 4096])
def test_ties_of_the_formula_are_the_kernels(rows):
    """How the codes and scales of random bfloat16 rows relate to a division by a number that is made a product with its inverse:
    they differ in the scale's last bit in some rows, and the kernel's are the quotients'."""
    from xeno_rt_b200.csrc import ops
    x = torch.randn(rows, 4096, generator=torch.Generator().manual_seed(rows)).to(DEV).bfloat16()
    codes, scales = ops.int8_rows(rows, 4096, DEV), torch.empty(rows, device=DEV)
    ops.quantize_rows(codes, scales, x)
    host = x.float().cpu().numpy()
    scale = np.abs(host).max(axis=1) / np.float32(127)
    assert np.array_equal(scales.cpu().numpy(), scale)
    assert np.array_equal(codes.cpu().numpy(), np.rint(host / scale[:, None]))
