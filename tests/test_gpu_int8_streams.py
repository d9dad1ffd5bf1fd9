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


@pytest.mark.parametrize("next_is_the_captures", [False, True])
@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
def test_a_first_call_inside_a_capture_reports_its_errors_too(monkeypatch, mode, next_is_the_captures):
    """The device's flag is made beside the capture: kernels of the graph get it, no replay clears it, and it is read as ever."""
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(5)).to(DEV)
    want, want_scales = ops.int8_rows(4, 64, DEV), torch.empty(4, device=DEV)
    ops.quantize_rows(want, want_scales, x)
    codes, scales = ops.int8_rows(4, 64, DEV), torch.empty(4, device=DEV)
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_error_flags", {})  # as in a process that has called nothing yet
    monkeypatch.setattr(ops, "_error_flags_at", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode=mode):
        own = torch.cuda.current_stream().cuda_stream
        if next_is_the_captures:  # the pool of streams is gone through until it gives the capture's again
            taken = [torch.cuda.Stream().cuda_stream for _ in range(128)]
            around = taken[::-1].index(taken[-1], 1)  # streams in the pool
            place = taken[::-1].index(own)  # how many came after the capture's
            for _ in range(around - 1 - place):
                torch.cuda.Stream()
        ops.quantize_rows(codes, scales, x)
        inside = ops._error_flag_pointer(0)
    flag = ops._error_flags[0]
    assert inside != 0 and inside == flag.data_ptr()
    graph.replay()
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)
    ops.check_error_flag(DEV)
    flag.fill_(7)  # as a kernel of the graph would
    graph.replay()
    with pytest.raises(KernelError, match="error 7"):
        ops.check_error_flag(DEV)
    ops.check_error_flag(DEV)
    del graph, codes, scales
    torch.cuda.empty_cache()
    assert ops.error_flag(DEV) is flag and int(flag) == 0
