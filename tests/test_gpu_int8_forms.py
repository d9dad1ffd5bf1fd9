"""8-bit products by every kernel, tile and plan that the launcher chooses from, against the formula in 64 bits.

``FORMS`` says of each size which it is (for 148 multiprocessors; tests/test_int8_forms.py holds the launcher to that).  Tolerance: the
sum is exact; 32-bit results have the sum's rounding, two products and at most two additions, five halves of 2^-23 of what is
added up; bfloat16 half of 2^-7 more."""
import functools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# (rows, outputs, inputs): kernel, what else is true of the plan
FORMS = {
    # pairs of blocks, 256 x 256: one tile a pair; several rounds of tiles (both accumulators, the ring's phases beyond
    # one turn), outputs that begin at no 16-byte boundary; rows beyond the first 4,096, which the walk takes as a second group
    (129, 10240, 4096): "pair256",
    (2500, 9000, 700): "pair256",
    (2500, 9003, 700): "pair256",
    (5000, 9000, 520): "pair256",
    (4200, 2999, 4000): "pair256",
    # pairs, 256 x 128: three rounds
    (200, 19000, 4096): "pair128",
    (200, 19003, 4096): "pair128",
    (400, 9500, 4096): "pair128",
    # single blocks, 128 x 256: two rounds
    (300, 19000, 4096): "single256",
    (300, 19001, 4096): "single256",
    (777, 10240, 4096): "single256",
    # single blocks, 128 x 128: several rounds, a second group of rows; few rows that go to tiles
    (9000, 700, 200): "single128",
    (1500, 9001, 333): "single128",
    (64, 2048, 128): "single128",
    (100, 102400, 640): "single128",
    (128, 20000, 4096): "single128",
    # few rows: tiles of one and of two MMAs (more than 128 weight rows), two blocks a multiprocessor, parts of K
    (8, 40000, 300): "few",
    (24, 40000, 4096): "few",
    (1, 19000, 1000): "few",
    (64, 28672, 4096): "few",
    (65, 37880, 4096): "few",
    (100, 25000, 4096): "few",
    (65, 10000, 14336): "few",
    (1, 600, 14336): "few",
    (7, 2048, 2048): "few",
    (80, 512, 768): "few",
    (128, 4096, 8192): "few",
}


def coded(rows, width, seed):
    from xeno_rt_b200.csrc import ops
    gen = torch.Generator(device=DEV).manual_seed(seed)
    codes = ops.int8_rows(rows, width, DEV)
    codes.copy_(torch.randint(-128, 128, (rows, width), generator=gen, device=DEV, dtype=torch.int8))
    return codes, torch.rand(rows, generator=gen, device=DEV) * 0.02 + 0.001


@functools.lru_cache(maxsize=1)
def case(m, n, k):
    """(codes, scales, weight, its scales, bias, the product in 64 bits)."""
    codes, scales = coded(m, k, 1)
    w, w_scales = coded(n, k, 2)
    bias = torch.randn(n, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    total = codes.double() @ w.double().t()
    total *= scales.double()[:, None]
    total *= w_scales.double()
    return codes, scales, w, w_scales, bias, total


def check(out, want, size):
    allowed = size * (5 * 2.0 ** -24)
    if out.dtype == torch.bfloat16:
        allowed = allowed + (want.abs() + allowed) * 2.0 ** -8
    assert bool(((out.double() - want).abs() <= allowed + 1e-40).all())


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("mode", ["float32", "bfloat16", "added"])
@pytest.mark.parametrize("m,n,k", list(FORMS))
def test_form(m, n, k, mode, biased):
    from xeno_rt_b200.csrc import ops
    codes, scales, w, w_scales, bias, total = case(m, n, k)
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    if sms == 148:
        assert ops.gemm_int8_plan(sms, m, n, k).kernel == FORMS[m, n, k]
    want, size = total, total.abs()
    if biased:
        want, size = want + bias.double(), size + bias.double().abs()
    if mode == "added":
        whole = torch.randn(m + 1, n, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
        before = whole.clone()
        ops.gemm_int8(whole[:m], codes, scales, w, w_scales, accumulate=True, bias=bias if biased else None, constant_weight=True)
        check(whole[:m], want + before[:m].double(), size + before[:m].double().abs())
        assert torch.equal(whole[m], before[m])
        return
    out = torch.full((m + 1, n), 5.0, dtype=getattr(torch, mode), device=DEV)
    ops.gemm_int8(out[:m], codes, scales, w, w_scales, bias=bias if biased else None)
    check(out[:m], want, size)
    assert bool((out[m] == 5.0).all())


@pytest.mark.parametrize("m,n,k", [(2500, 9000, 700), (200, 19000, 4096), (300, 19001, 4096), (1500, 9001, 333), (64, 28672, 4096)])
def test_forms_into_strided_rows_and_again(m, n, k):
    """Rows with room between them (at 16 bytes, and not), which stays as it was; and the same bits every time."""
    from xeno_rt_b200.csrc import ops
    codes, scales, w, w_scales, _, total = case(m, n, k)
    first = None
    for room in (8, 5):
        whole = torch.full((m, n + room), 5.0, device=DEV)
        for _ in range(3):
            ops.gemm_int8(whole[:, :n], codes, scales, w, w_scales)
            first = whole[:, :n].clone() if first is None else first
            assert torch.equal(whole[:, :n], first)
        assert bool((whole[:, n:] == 5.0).all())
    check(first, total, total.abs())
