"""Who may hold tensor memory while somebody else waits for it (reads the kernels' sources and plans: no GPU)."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xeno-rt_b200", "csrc")


def _allocating_kernels():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith(".cu"):
            with open(os.path.join(CSRC, name)) as fh:
                text = fh.read()
            for i, body in enumerate(re.split(r"\b__global__\b", text)[1:]):
                if "tcgen05.alloc" in body:
                    yield pytest.param(body, id=f"{name}:{i}")


@pytest.mark.parametrize("body", list(_allocating_kernels()))
def test_a_successor_may_be_launched_only_when_the_columns_are_taken(body):
    """A successor's block that is launched early waits for this kernel as a whole: were it to get the columns that a block of this
    one still waits for, neither would go on."""
    triggers = [m.start() for m in re.finditer(r"pdl_trigger\(\)", body)]
    allocations = [m.start() for m in re.finditer(r"tcgen05\.alloc\.", body)]
    assert not triggers or min(triggers) > max(allocations)


def test_blocks_that_fit_a_multiprocessor_find_their_columns():
    """The 8-bit products of few rows: shared memory in proportion to the columns, for a device of 148 multiprocessors."""
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops
    try:
        ops.library()  # the arithmetic lives beside the kernel it describes; building needs nvcc, not a GPU
    except KernelError as exc:
        pytest.skip(f"the kernel library cannot be built here: {exc}")
    seen = set()
    for m in (1, 16, 17, 33, 48, 49, 64, 65, 80, 96, 97, 112, 128):
        for n in (1, 32, 72, 515, 1024, 2048, 4096, 6144, 10240, 19000, 28672, 51200, 102400):
            for k in (1, 128, 129, 300, 512, 1000, 1024, 2048, 4096, 14336, 131071):
                plan = ops.gemm_int8_plan(148, m, n, k)
                if plan.kernel == "few":
                    seen.add((plan.columns, plan.splits))
                    assert (plan.shared_bytes + 1024) * 512 >= plan.columns * 228 * 1024
                    assert plan.shared_bytes <= 227 * 1024
    assert {columns for columns, _ in seen} == {32, 64, 128, 256} and {splits for _, splits in seen} == {1, 2, 3, 4}


_DECODE = r"""
#include <cuda_runtime.h>
#include <cstdio>
inline cudaError_t no_device(int*) { return cudaErrorNoDevice; }
#define cudaGetDevice no_device
#include "gemm_decode_tcgen05.cu"
namespace xrt { const Tuning& tuning() { static const Tuning t; return t; } }
int main() {
  int bad = 0, most = 0, plans = 0;
  for (int mode = 0; mode < 3; ++mode)
    for (int m = 1; m <= 128; m += m < 16 ? 5 : 16)
      for (int n : {128, 1000, 4096, 14336, 28672, 128256})
        for (int k : {64, 512, 4096, 14336}) {
          xrt::DecodeGemmShape shape;
          int smem = 0, blocks = 0;
          if (xrt::plan_decode_gemm(m, n, k, n, mode, mode == 2 ? n : 0, 148, &shape, &smem, &blocks) != XRT_OK) continue;
          ++plans;
          if (shape.tmem_cols > most) most = shape.tmem_cols;
          if ((smem + 1024) * 512ll < shape.tmem_cols * 228ll * 1024 || smem > 227 * 1024) ++bad;
        }
  printf("%d %d %d", plans, bad, most);
  return 0;
}
"""


def test_the_same_of_the_products_of_few_rows_in_bfloat16(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    (tmp_path / "main.cu").write_text(_DECODE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O0", "-Xcicc", "-O0", "-Xptxas", "-O0", "-std=c++17", "-I", CSRC,
                    "-o", str(tmp_path / "main"), str(tmp_path / "main.cu")], check=True, capture_output=True, text=True)
    plans, bad, most = map(int, subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout.split())
    assert plans > 200 and most == 512 and bad == 0


_SIZES = r"""
#include <cuda_runtime.h>
#include <cstdio>
#include "gemm_tcgen05.cu"
#include "gemm_int8.cu"
namespace xrt { const Tuning& tuning() { static const Tuning t; return t; } }
int main() {
  printf("%d %d %d", xrt::TcShape<true>::SMEM, xrt::Int8Shape<true, 256>::SMEM, xrt::Int8Shape<true, 128>::SMEM);
  return 0;
}
"""


def test_no_block_with_tensor_memory_fits_beside_a_pair_that_has_all_of_it(tmp_path):
    """Pairs of blocks take 512 columns in one multiprocessor and wait for as many in another: a block that fitted beside them could
    hold what they wait for."""
    from xeno_rt_b200.core import KernelError
    from xeno_rt_b200.csrc import ops
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    try:
        ops.library()
    except KernelError as exc:
        pytest.skip(f"the kernel library cannot be built here: {exc}")
    (tmp_path / "main.cu").write_text(_SIZES)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O0", "-Xcicc", "-O0", "-Xptxas", "-O0", "-std=c++17", "-I", CSRC,
                    "-o", str(tmp_path / "main"), str(tmp_path / "main.cu")], check=True, capture_output=True, text=True)
    bf16, all_columns, half = map(int, subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout.split())
    least = min(p.shared_bytes for p in (ops.gemm_int8_plan(148, m, n, k) for m in (1, 16, 64, 128) for n in (1, 8, 600, 6144, 40000)
                                         for k in (1, 128, 300, 4096)) if p.kernel == "few")
    for pair in (bf16, all_columns):
        assert pair + 1024 + least + 1024 > 228 * 1024
    assert (half + 1024) * 512 >= 256 * 228 * 1024
