"""Weights that were laid out in 8 bits right before the product that reads them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows", [1, 8, 64, 300])
@pytest.mark.parametrize("rows_first", [False, True])
def test_a_product_right_after_its_matrix_was_made(rows, rows_first):
    """Products of few rows read a constant weight ahead of their wait for the kernels before them: a matrix is one only once
    its codes are written."""
    from xeno_rt_b200.csrc import ops
    from xeno_rt_b200.parts.int8 import Int8Matrix, Int8Rows
    from xeno_rt_b200.parts.linear import linear
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, 4096, generator=gen, device=DEV)
    weights = [torch.randn(16384, 4096, generator=gen, device=DEV) for _ in range(4)]
    want = []
    for w in weights:
        codes, scales = ops.int8_rows(16384, 4096, DEV), torch.empty(16384, device=DEV)
        ops.quantize_rows(codes, scales, w)
        h = Int8Rows.of(x)
        out = torch.empty(rows, 16384, device=DEV)
        torch.cuda.synchronize()
        ops.gemm_int8(out, h.codes, h.scales, codes, scales)
        want.append(out)
        codes.fill_(0)  # what a reader of memory that is used again would see
    del codes
    torch.cuda.synchronize()
    for w, right in zip(weights, want):
        h = Int8Rows.of(x) if rows_first else x
        out = linear(h, Int8Matrix.of(w))
        assert torch.equal(out, right)


def test_a_matrix_is_not_laid_out_inside_a_capture():
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops
    from xeno_rt_b200.parts.int8 import Int8Matrix, product
    w = torch.randn(256, 128, generator=torch.Generator().manual_seed(1)).to(DEV)
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(2)).to(DEV)
    matrix, out = Int8Matrix.of(w), torch.empty(4, 256, device=DEV)
    assert matrix.constant and matrix[:16].constant and not Int8Matrix(matrix.codes, matrix.scales).constant
    product(out, x, matrix, False)
    want, graph = out.clone(), torch.cuda.CUDAGraph()
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(KernelError, match="capture"):
            Int8Matrix.of(w)
        product(out, x, matrix, False)  # which the refusal left as it was
    graph.replay()
    assert torch.equal(out, want)


def test_memory_while_a_model_is_loaded(tmp_path):
    """The whole model in the compute dtype, then part by part in 8 bits: the peak is the former and no more than the codes of
    one layer, whose matrices are given up when all of its parts are laid out; what is left is less."""
    from helpers import CONFIGS
    from xeno_rt_b200 import write_random_model
    from xeno_rt_b200.engine import Model
    raw = dict(CONFIGS["tiny-wide"][0], hidden_size=1024, intermediate_size=4096, num_hidden_layers=6)
    folder = str(tmp_path / "m")
    write_random_model(folder, raw, 1, "bfloat16")
    left, peak = {}, {}
    for weights in (None, "int8"):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        model = Model.load(folder, dtype="bfloat16", weights=weights)
        torch.cuda.synchronize()
        left[weights], peak[weights] = torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before
        del model
    layer = 3 * 1024 * 4096 + 1024 * (raw["num_attention_heads"] + raw["num_key_value_heads"]) * raw["head_dim"] * 2  # bytes of codes
    assert left["int8"] < left[None] - 0.9 * 6 * layer
    assert peak["int8"] <= peak[None] + 1.1 * layer
