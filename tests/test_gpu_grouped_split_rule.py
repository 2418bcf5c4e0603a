"""More columns of the same few rows never take much less time: K is split over no more clusters than the GPU holds."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200.kernels import grouped_gemm  # noqa: E402
from tests.timing_helpers import device_us  # noqa: E402


def _us(rows, tiles, k=4096):
    """Device time of a call on 128 * tiles columns."""
    n = 128 * tiles
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")

    def operands():
        return (torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda"),
                torch.zeros((1, k, n), dtype=torch.bfloat16, device="cuda"), offsets,
                torch.empty((rows, n), dtype=torch.bfloat16, device="cuda"))

    return device_us(grouped_gemm, operands, 2 * k * n)


# The later count takes the next smaller cluster in any case; a second round of clusters costs 1.3 to 1.4 times its time.
@pytest.mark.parametrize("rows, tiles, later", [(50, 16, 19), (50, 18, 19), (50, 34, 38), (50, 37, 38), (3, 37, 38),
                                                (3, 74, 75)])
def test_fewer_tiles_take_no_longer(rows, tiles, later):
    assert min(_us(rows, tiles) for _ in range(2)) <= 1.12 * max(_us(rows, later) for _ in range(2))
