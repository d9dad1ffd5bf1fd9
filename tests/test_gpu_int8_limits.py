"""The largest calls of the 8-bit operators: offsets beyond 32 bits, the longest rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from xeno_rt_b200.csrc import ops as o
    return o


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("less than 40 GB are free")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,width", [(1, 2 ** 31 - 8192), (1, 2 ** 31 - 8199), (3, 2 ** 30 + 8), (70001, 65536)])
def test_rows(rows, width):
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    at = [0, 7, 8191, 8192, width // 2 + 1, width - 8193, width - 9, width - 1]
    values = torch.tensor([1, 2, 3, 5, 6, 7, 8, 8], device=DEV, dtype=torch.float64)  # none lies between two codes
    some = sorted({0, rows // 2, rows - 1})
    for r in some:
        x[r, at] = values.bfloat16() * (r % 5 + 1)
    codes = torch.full((rows, width), 55, dtype=torch.int8, device=DEV)
    scales = torch.empty(rows, device=DEV)
    ops().quantize_rows(codes, scales, x)
    for r in some:
        assert torch.equal(codes[r, at].double(), (values * 127 / 8).round()) and scales[r].item() == pytest.approx(8 * (r % 5 + 1) / 127, rel=2.0 ** -23)
    assert int(sum(torch.count_nonzero(part) for part in codes.view(-1).split(2 ** 30))) == 8 * len(some)


@pytest.mark.parametrize("m", [1, 200])
def test_products_with_weights_beyond_32_bits(m):
    """2^32 bytes of weights: the last rows' sums against the formula's."""
    o = ops()
    n, k = 33000, 131071
    w = torch.randint(-128, 128, (n, 131072), dtype=torch.int8, device=DEV)[:, :k]
    codes = torch.randint(-128, 128, (m, 131072), dtype=torch.int8, device=DEV)[:, :k]
    ones = torch.ones(n, device=DEV)
    out = torch.empty(m, n, device=DEV)
    o.gemm_int8(out, codes, ones[:m], w, ones)
    for lo in (0, 16380, 32744):
        want = codes.double() @ w[lo:lo + 256].double().t()
        assert torch.equal(out[:, lo:lo + 256], want.float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [32768, 32769])
def test_products_with_outputs_beyond_32_bits(n, dtype):
    o = ops()
    m, k = 70001, 16
    codes = torch.randint(-128, 128, (m, k), dtype=torch.int8, device=DEV)
    w = torch.randint(-128, 128, (n, k), dtype=torch.int8, device=DEV)
    out = torch.zeros(m, n, dtype=dtype, device=DEV)
    o.gemm_int8(out, codes, torch.ones(m, device=DEV), w, torch.ones(n, device=DEV))
    for lo in (0, 65400, m - 256):
        want = codes[lo:lo + 256].double() @ w.double().t()
        assert torch.equal(out[lo:lo + 256], want.to(dtype))
