"""Rows that begin anywhere on their way to one or two experts: how much longer they take than aligned ones."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200.kernels import expert_dispatch  # noqa: E402
from tests.timing_helpers import device_us  # noqa: E402


def _us(tokens, choices, width):
    def operands():
        slots = torch.randperm(tokens * choices, device="cuda").view(tokens, choices).to(torch.int32)
        return (torch.zeros((tokens, width), dtype=torch.bfloat16, device="cuda"), slots,
                torch.empty((tokens * choices, width), dtype=torch.bfloat16, device="cuda"))

    return device_us(expert_dispatch, operands, 2 * tokens * (1 + choices) * width)


# us: 16384 tokens of one and two rows, 4096 wide 48 and 65, 4095 wide 75 and 103 (slots four at once: 108 and 126); 4109
# tokens of 8 rows, 2048 wide 25.2, 2046 wide 31 (weights read ahead of the look at the slot: 36).
@pytest.mark.parametrize("tokens, choices, width, aligned, share", [(16384, 1, 4095, 4096, 1.9), (16384, 2, 4095, 4096, 1.76),
                                                                    (4109, 8, 2046, 2048, 1.32)])
def test_rows_that_begin_anywhere_take_little_longer(tokens, choices, width, aligned, share):
    assert min(_us(tokens, choices, width) for _ in range(2)) <= share * max(_us(tokens, choices, aligned) for _ in range(2))
