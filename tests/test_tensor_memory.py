"""Who may hold tensor memory while somebody else waits for it (reads the kernels' sources and plans: no GPU)."""
import os
import re

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
