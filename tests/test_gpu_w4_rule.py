"""Rows of a long k that do not fit at once: as many passes over the 4-bit weights with the narrower products."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200.kernels import gemv_w4  # noqa: E402
from tests.timing_helpers import device_us  # noqa: E402


def _us(rows, n, k):
    def operands():
        return (torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda"),
                torch.zeros((n, k // 2), dtype=torch.uint8, device="cuda"),
                torch.zeros((n, k // 128), dtype=torch.bfloat16, device="cuda"),
                torch.empty((rows, n), dtype=torch.bfloat16, device="cuda"))

    return device_us(gemv_w4, operands, n * k // 2)


# 16 rows take two passes at all of these k, at 8192 with the narrower products in any case; with the wider ones the
# shorter k took 0.91 and 1.03 of its time.
@pytest.mark.parametrize("k, share", [(4608, 0.75), (6144, 0.9)])
def test_a_shorter_k_takes_less_time(k, share):
    assert min(_us(16, 16384, k) for _ in range(2)) <= share * max(_us(16, 16384, 8192) for _ in range(2))
