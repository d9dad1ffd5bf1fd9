"""What lies beside the rows that an 8-bit product writes stays as it was, to the bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("mode", ["float32", "bfloat16", "added"])
@pytest.mark.parametrize("more", range(8))
@pytest.mark.parametrize("m,n,k", [(3, 640, 96), (200, 640, 256), (384, 6312, 128), (300, 19000, 256), (200, 19000, 512), (1300, 9000, 512)])
def test_rows_that_begin_but_do_not_end_every_16_bytes(m, n, k, more, mode):
    """Rows 16 bytes apart of any number of columns, in a buffer of minus zeros, NaNs and other numbers."""
    from xeno_rt_b200.csrc import ops
    dtype = torch.bfloat16 if mode == "bfloat16" else torch.float32
    ints = torch.int16 if dtype == torch.bfloat16 else torch.int32
    n, ld = n + more, n + 16
    codes, w = ops.int8_rows(m, k, DEV), ops.int8_rows(n, k, DEV)
    gen = torch.Generator(device=DEV).manual_seed(n)
    codes.copy_(torch.randint(-9, 10, (m, k), generator=gen, device=DEV))
    w.copy_(torch.randint(-9, 10, (n, k), generator=gen, device=DEV))
    whole = torch.full((m * ld + 64,), -0.0, dtype=dtype, device=DEV)
    whole[1::3] = float("nan")
    whole[2::5] = 5.0
    rows = whole[32:32 + m * ld].view(m, ld)
    rows[:, :n] = 3.0
    before = whole.clone()
    ops.gemm_int8(rows[:, :n], codes, torch.ones(m, device=DEV), w, torch.ones(n, device=DEV), accumulate=mode == "added")
    total = codes.double() @ w.double().t()  # whole numbers below 2^24
    assert torch.equal(rows[:, :n], (total + 3 if mode == "added" else total).to(dtype))
    before[32:32 + m * ld].view(m, ld)[:, :n] = rows[:, :n]
    assert torch.equal(whole.view(ints), before.view(ints))
