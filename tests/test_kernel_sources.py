"""Orders inside the kernels that no run on one GPU can show, read from their sources."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "teamredbench_b200" / "csrc"
ALLOC = re.compile(r"\btmem_alloc(?:_pair)?\(")


def _kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for start, end in zip(starts, starts[1:]):
            body = text[start:end]
            name = re.search(r"(\w+)\s*\(\s*(?:const|uint|void|int|float)", body)
            yield f"{path.name}:{name.group(1) if name else start}", body


KERNELS = dict(_kernels())
DEPENDENTS = [k for k, body in KERNELS.items() if ALLOC.search(body) and "grid_launch_dependents()" in body]


def test_kernels_are_found():
    for name in ("grouped_gemm_kernel", "grouped_split_kernel", "grouped_wgrad_kernel"):
        assert f"gemm_grouped.cu:{name}" in DEPENDENTS
    assert len(DEPENDENTS) >= 7


@pytest.mark.parametrize("kernel", DEPENDENTS)
def test_tensor_memory_is_allocated_before_the_next_grid_may_start(kernel):
    """One thread's grid_launch_dependents counts for its whole block.  A following grid may then take tensor memory on
    the same SM and keep it until this grid is done, so a block that had still to allocate might never get any: the
    allocation comes first, and a barrier of the block stands between the two."""
    body = KERNELS[kernel]
    allocated = max(m.end() for m in ALLOC.finditer(body))
    launch = body.index("grid_launch_dependents()")
    assert allocated < launch
    assert "__syncthreads()" in body[allocated:launch]
