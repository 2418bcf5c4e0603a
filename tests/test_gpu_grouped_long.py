"""Weight gradient of calls that last longer than any one step of a pipeline may."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import grouped_gemm_wgrad  # noqa: E402


def test_waits_are_for_a_stage_not_for_the_call():
    """A group of 2^29 rows is one tile of 4.2 million stages, more than two seconds on one pair of blocks; the last
    group's tile is the same pair's next one, and the only one whose last stage has rows to clear.  Neither the warp
    that clears them nor the ones that read the results out may take the time before their turn for a hang."""
    long_rows = 1 << 29
    groups = torch.cuda.get_device_properties(0).multi_processor_count // 2 + 1
    rows = long_rows + 5
    offsets = torch.full((groups + 1,), long_rows, dtype=torch.int32, device="cuda")
    offsets[0], offsets[-1] = 0, rows
    # All zeros but for a few rows of small whole numbers, so that every sum is exact.
    a = torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda")
    grad = torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda")
    places = torch.tensor([0, 3, 1 << 20, (1 << 28) + 77, long_rows - 1] + list(range(long_rows, rows)), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    a[places] = torch.randint(-3, 4, (10, 8), generator=gen, device="cuda").bfloat16()
    grad[places] = torch.randint(-3, 4, (10, 8), generator=gen, device="cuda").bfloat16()
    out = torch.full((groups, 8, 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    assert _native.device_error(0, clear=True) == 0
    grouped_gemm_wgrad(a, grad, offsets, out)
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0
    x, g = a[places].double(), grad[places].double()
    assert torch.equal(out[0].double(), x[:5].T @ g[:5])
    assert torch.equal(out[-1].double(), x[5:].T @ g[5:])
    assert not out[1:-1].any()
