"""GPU tests of expert_sort at every size of its cluster (1, 4, 8 and 16 CTAs), with several experts at each."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200.kernels import expert_sort  # noqa: E402


# Groups of 32 choices around the borders: up to 64 groups one CTA, to 256 four, to 512 eight, then sixteen, whose warps
# keep up to eight groups in registers (4096 groups), and work through more in turns.
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens, choices", [(2048, 1), (2049, 1), (8192, 1), (8193, 1), (2049, 4), (10007, 1), (8192, 2),
                                             (16385, 1), (16384, 8), (131073, 1), (150001, 7)])
@pytest.mark.parametrize("experts, outside", [(8, 0.0), (8, 0.4), (33, 0.1), (256, 0.0), (1024, 0.2)])
def test_sort_at_every_size_of_the_cluster(dtype, tokens, choices, experts, outside):
    g = torch.Generator(device="cuda").manual_seed(tokens + experts)
    ids = torch.randint(0, experts, (tokens, choices), device="cuda", generator=g)
    gone = torch.rand(ids.shape, device="cuda", generator=g) < outside
    ids = torch.where(gone, torch.where(torch.rand(ids.shape, device="cuda", generator=g) < 0.5, -1, experts), ids)
    flat = ids.reshape(-1)
    here = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(here, flat, experts), stable=True).indices[:int(here.sum())]
    want = torch.full_like(flat, -1)
    want[order] = torch.arange(order.numel(), device="cuda")
    counts = torch.bincount(flat[here], minlength=experts)
    offsets, slots = expert_sort(ids.to(dtype), torch.full((experts + 1,), -7, device="cuda", dtype=torch.int32),
                                 torch.full(ids.shape, -7, device="cuda", dtype=torch.int32))
    assert torch.equal(slots.reshape(-1).long(), want)
    assert offsets[0] == 0 and torch.equal(offsets[1:].long(), torch.cumsum(counts, 0))
