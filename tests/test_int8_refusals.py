"""Calls of the 8-bit operators that are refused before any device is asked."""
import pytest
import torch


def ops():
    from xeno_rt_b200.csrc import ops as o
    return o


def refused(match, call, *args, **options):
    from xeno_rt_b200.core import KernelError
    with pytest.raises(KernelError, match=match):
        call(*args, **options)


def test_rows_begin_every_16_bytes():
    for width in (1, 15, 16, 17, 4096):
        codes = ops().int8_rows(3, width, "cpu")
        assert codes.shape == (3, width) and codes.stride(0) % 16 == 0 and codes.stride(1) == 1


def test_shapes_and_types():
    o = ops()
    x, codes, scales = torch.zeros(3, 20), o.int8_rows(3, 20, "cpu"), torch.zeros(3)
    refused("int8", o.quantize_rows, torch.zeros(3, 20), scales, x)
    refused("int8", o.quantize_rows, o.int8_rows(3, 21, "cpu"), scales, x)
    refused("contiguous", o.quantize_rows, o.int8_rows(20, 3, "cpu").t(), scales, x)
    refused("contiguous", o.quantize_rows, o.int8_rows(1, 20, "cpu").expand(3, 20), scales, x)
    refused("scales", o.quantize_rows, codes, torch.zeros(4), x)
    refused("scales", o.quantize_rows, codes, scales.double(), x)
    refused(r"\[rows, width\]", o.quantize_rows, codes, scales, torch.zeros(60))
    refused("CUDA", o.quantize_rows, codes, scales, x)
    refused("gate_up", o.swiglu_int8, codes, scales, torch.zeros(3, 41))
    refused("one bias", o.swiglu_int8, codes, scales, torch.zeros(3, 40), o.Gate("silu", bias=torch.zeros(39)))
    refused("activation", o.swiglu_int8, codes, scales, torch.zeros(3, 40), "relu")
    refused("no add", o.rmsnorm_int8, codes, scales, x, torch.ones(20), 1e-5, out=x)
    refused("weight", o.rmsnorm_int8, codes, scales, x, torch.ones(21), 1e-5)
    refused("shape of x", o.rmsnorm_int8, codes, scales, x, torch.ones(20), 1e-5, add=torch.zeros(3, 21))
    refused("shape of x", o.rmsnorm_int8, codes, scales, x, torch.ones(20), 1e-5, add=x, out=torch.zeros(2, 20))


def test_products():
    o = ops()
    codes, scales, w, w_scales = o.int8_rows(3, 20, "cpu"), torch.zeros(3), o.int8_rows(5, 20, "cpu"), torch.zeros(5)
    out = torch.zeros(3, 5)
    refused("do not fit", o.gemm_int8, out, codes, scales, o.int8_rows(5, 21, "cpu"), w_scales)
    refused("16 bytes", o.gemm_int8, out, torch.zeros(3, 20, dtype=torch.int8), scales, w, w_scales)
    refused("16 bytes", o.gemm_int8, out, codes, scales, torch.zeros(5, 20, dtype=torch.int8), w_scales)
    shifted = torch.zeros(5 * 32 + 1, dtype=torch.int8)[1:].view(5, 32)[:, :20]
    refused("16 bytes", o.gemm_int8, out, codes, scales, shifted, w_scales)
    refused("contiguous", o.gemm_int8, out.t().contiguous().t(), codes, scales, w, w_scales)
    refused("out must be", o.gemm_int8, torch.zeros(3, 6), codes, scales, w, w_scales)
    refused("added into", o.gemm_int8, out.bfloat16(), codes, scales, w, w_scales, accumulate=True)
    refused("float32", o.gemm_int8, out, codes, scales, w, torch.zeros(4))
    refused("float32", o.gemm_int8, out, codes, scales, w, w_scales, bias=torch.zeros(5, dtype=torch.bfloat16))
    too_long = o.INT8_MAX_INPUTS + 1
    refused("32 bits", o.gemm_int8, out, o.int8_rows(3, too_long, "cpu"), scales, o.int8_rows(5, too_long, "cpu"), w_scales)


def test_models_that_hold_no_8_bit_weights():
    from helpers import TINY_QWEN3
    from xeno_rt_b200.config import config_from_dict
    from xeno_rt_b200.core import ConfigError, Unsupported
    from xeno_rt_b200.engine.model import check_weights_format
    from zivovik_cases import CASE_MIXED as other

    def spec(raw):
        arch, config = config_from_dict(raw)
        return arch.build_spec(config)

    check_weights_format(spec(TINY_QWEN3), None)
    check_weights_format(spec(TINY_QWEN3), "int8")
    with pytest.raises(ConfigError, match="int4"):
        check_weights_format(spec(TINY_QWEN3), "int4")
    with pytest.raises(Unsupported, match="8-bit weights"):
        check_weights_format(spec(other), "int8")


def test_the_command_takes_the_option():
    from xeno_rt_b200.cli import build_parser
    args = build_parser().parse_args(["generate", "--model", "m", "--prompt-ids", "1", "--weights", "int8"])
    assert args.weights == "int8"
    assert build_parser().parse_args(["generate", "--model", "m", "--prompt-ids", "1"]).weights is None
