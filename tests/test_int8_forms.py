"""Which kernel takes an 8-bit product (host arithmetic, for a device of 148 multiprocessors)."""
import pytest


@pytest.fixture(scope="module")
def plan():
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops
    try:
        ops.library()  # the arithmetic lives beside the kernel it describes; building needs nvcc, not a GPU
    except KernelError as exc:
        pytest.skip(f"the kernel library cannot be built here: {exc}")
    return lambda *size: ops.gemm_int8_plan(148, *size)


def test_the_sizes_that_are_tested_on_the_device_reach_every_form(plan):
    from test_gpu_int8_forms import FORMS
    plans = {size: plan(*size) for size in FORMS}
    assert {size: p.kernel for size, p in plans.items()} == FORMS
    assert set(FORMS.values()) == {"pair256", "pair128", "single256", "single128", "few"}
    few = [p for p in plans.values() if p.kernel == "few"]
    assert {p.columns for p in few if p.rows > 128} >= {32, 64, 256}  # two MMAs, the second's sums beside the first's
    assert any(p.blocks > 148 for p in few)  # two blocks a multiprocessor
    assert {p.splits for p in few} == {1, 2, 3, 4}

    def rounds(kernel, rows, columns, at_once):
        return max(-(-m // rows) * -(-n // columns) / at_once for (m, n, k), p in plans.items() if p.kernel == kernel)

    # persistent blocks that walk several tiles
    assert rounds("pair256", 256, 256, 74) > 4 and rounds("pair128", 256, 128, 74) > 2
    assert rounds("single256", 128, 256, 148) > 1 and rounds("single128", 128, 128, 148) > 4


def test_no_size_is_without_a_plan(plan):
    for m in (1, 2, 15, 16, 17, 48, 49, 100, 128, 129, 256, 257, 1000, 8192):
        for n in (1, 7, 64, 515, 6144, 18944, 18945, 37888, 37889, 102400):
            for k in (1, 16, 127, 128, 129, 1000, 4096, 131071):
                p = plan(m, n, k)
                if p.kernel == "few":
                    assert m <= 128 and 8 <= p.rows <= 256 and p.rows % 8 == 0 and 1 <= p.splits <= 4
                    assert p.blocks == -(-n // p.rows) * p.splits and p.blocks // p.splits < 65536 and p.shared_bytes <= 227 * 1024
