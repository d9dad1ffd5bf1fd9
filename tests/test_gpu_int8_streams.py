"""8-bit products beside one another: on several streams and on few multiprocessors' worth of tensor memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def coded(rows, width, seed):
    from xeno_rt_b200.csrc import ops
    codes = ops.int8_rows(rows, width, DEV)
    codes.copy_(torch.randint(-128, 128, (rows, width), generator=torch.Generator().manual_seed(seed)).to(DEV))
    return codes, torch.rand(rows, generator=torch.Generator().manual_seed(seed + 1)).to(DEV) * 0.02 + 0.001


@pytest.mark.parametrize("m,n,k", [(80, 512, 768), (96, 512, 1024), (128, 1024, 1024)])
def test_chains_of_short_products_on_eight_streams(m, n, k):
    """Parts of K in clusters, 128 columns of tensor memory a block: five such blocks would have more columns than a
    multiprocessor.  Every result is that of the product alone."""
    from xeno_rt_b200.csrc import ops
    plan = ops.gemm_int8_plan(torch.cuda.get_device_properties(DEV).multi_processor_count, m, n, k)
    assert plan.columns == 128 and plan.splits > 1
    cases = [(coded(m, k, 10 + i), coded(n, k, 40 + i)) for i in range(8)]
    want = []
    for (c, s), (w, ws) in cases:
        out = torch.empty(m, n, device=DEV)
        ops.gemm_int8(out, c, s, w, ws)
        want.append(out)
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty(m, n, device=DEV) for _ in range(12)] for _ in cases]
    torch.cuda.synchronize()
    for turn in range(12):
        for ((c, s), (w, ws)), stream, out in zip(cases, streams, outs):
            with torch.cuda.stream(stream):
                ops.gemm_int8(out[turn], c, s, w, ws, constant_weight=turn % 2 == 1)
    torch.cuda.synchronize()
    ops.check_error_flag(DEV)
    for one, got in zip(want, outs):
        assert all(torch.equal(one, out) for out in got)
