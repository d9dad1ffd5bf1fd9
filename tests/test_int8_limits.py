"""The largest calls of the 8-bit operators: what is refused, without a device."""
import pytest
import torch


def test_sizes_that_pass_the_kernels_counters_are_refused():
    """A counter of 32 bits that is stepped on beyond the last element would come back below zero."""
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops as o

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="meta")

    calls = []
    for size in (o.INT8_MAX_SIZE + 1, 2 ** 31 - 1, 2 ** 31, 2 ** 32):
        wide, tall = empty(1, size, dtype=torch.int8), empty(size, 16, dtype=torch.int8)
        calls += [
            lambda wide=wide, size=size: o.quantize_rows(wide, empty(1), empty(1, size)),
            lambda wide=wide, size=size: o.swiglu_int8(wide, empty(1), empty(1, 2 * size)),
            lambda wide=wide, size=size: o.rmsnorm_int8(wide, empty(1), empty(1, size), empty(size), 1e-5),
            lambda tall=tall, size=size: o.quantize_rows(tall, empty(size), empty(size, 16)),
            lambda tall=tall, size=size: o.gemm_int8(empty(size, 1), tall, empty(size), empty(1, 16, dtype=torch.int8), empty(1)),
            lambda tall=tall, size=size: o.gemm_int8(empty(1, size), empty(1, 16, dtype=torch.int8), empty(1), tall, empty(size)),
        ]
    for call in calls:
        with pytest.raises(KernelError, match="too large"):
            call()


def test_the_launchers_refuse_them_too():
    """Plans are host arithmetic; a launcher that is called past the Python side sees the same limit."""
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops as o
    try:
        o.library()
    except KernelError as exc:
        pytest.skip(f"the kernel library cannot be built here: {exc}")
    assert o.gemm_int8_plan(148, o.INT8_MAX_SIZE, 1, 16).kernel != "few" and o.gemm_int8_plan(148, 1, o.INT8_MAX_SIZE, 16).kernel != "few"
    for m, n, k in ((o.INT8_MAX_SIZE + 1, 1, 16), (1, o.INT8_MAX_SIZE + 1, 16), (1, 1, o.INT8_MAX_INPUTS + 1)):
        with pytest.raises(KernelError):
            o.gemm_int8_plan(148, m, n, k)
    # (nothing is launched: the arguments are refused before)
    for n, width in ((o.INT8_MAX_SIZE + 1, 16), (1, o.INT8_MAX_SIZE + 1)):
        call = o._pack_int8_rows(16, 16, 16, 0, 0, 0, 0, 0, n, width, max(width, 16), 0, 0, 0, 0, 0, 0.0)
        assert o.library().xrt_quantize_rows(call, 0) == -1
    for m, n in ((o.INT8_MAX_SIZE + 1, 1), (1, o.INT8_MAX_SIZE + 1)):
        call = o._pack_int8_product(16, 16, 16, 16, 16, 0, 0, m, n, 16, 16, 16, n, 0, 0, 0)
        assert o.library().xrt_gemm_int8(call, 0) == -1


def test_the_option_says_that_the_products_inputs_are_rounded_too(capsys):
    from xeno_rt_b200.cli import build_parser
    from xeno_rt_b200.engine.runtime import Runtime
    with pytest.raises(SystemExit):
        build_parser().parse_args(["generate", "--help"])
    said = " ".join(capsys.readouterr().out.split())
    assert "round the inputs of their products to 8 bits too" in said
    assert "inputs of their products" in " ".join(Runtime.load.__doc__.split())
