"""Rows and results behind 2^31 elements, and calls at the ends of the kernels' own sizes."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import (  # noqa: E402
    dequantize_fp4, expert_combine, expert_combine_grad, expert_dispatch, expert_sort, gemm_fp4, quantize_fp4)
from tests.fp4_helpers import check, operand, product, values  # noqa: E402

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def no_device_error():
    assert _native.device_error(0, clear=True) == 0
    torch.manual_seed(11)
    yield
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0
    torch.cuda.empty_cache()


def _randn(shape, seed, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("width", [32768, 32767])
def test_rows_behind_2_31_elements(width):
    rows = 2 ** 31 // width + 40
    big = torch.zeros(rows, width, device="cuda", dtype=BF16)
    x, w = _randn((6, width), 1), _randn((6, 2), 2, torch.float32)
    slots = torch.randperm(30, device="cuda")[:12].view(6, 2).to(torch.int32) + (rows - 30)
    slots[0, 0], slots[5, 1] = 0, -1
    here = slots >= 0
    expert_dispatch(x, slots, big)
    want = x.unsqueeze(1).expand(-1, 2, -1)[here]
    assert torch.equal(big[slots[here].long()], want)
    out = torch.empty_like(x)
    expert_combine(big, slots, out)
    assert torch.equal(out, (x.float() * here.sum(1, keepdim=True)).to(BF16))
    grad_y, grad_w = torch.zeros_like(big), torch.empty_like(w)
    expert_combine_grad(x, big, slots, w, grad_y, grad_w)
    want_w = torch.where(here, (x.double() ** 2).sum(1, keepdim=True), 0.0)
    # sums of `width` products of one sign in fp32: each add drops at most 2^-24 of what is there
    assert ((grad_w.double() - want_w).abs() <= width * 2.0 ** -24 * want_w).all()
    want_y = (x.unsqueeze(1).float() * w.unsqueeze(-1)).to(BF16)[here]
    assert torch.equal(grad_y[slots[here].long()], want_y)


def test_codes_and_values_behind_2_31():
    k = 32768
    rows = 2 ** 32 // k + 20  # codes behind 2^31 bytes
    x = _randn((5, k), 1)
    q = torch.zeros(rows, k // 2, device="cuda", dtype=torch.uint8)
    scales = torch.zeros(rows, k // 32, device="cuda", dtype=torch.uint8)
    slots = torch.tensor([[rows - 1], [rows - 7], [3], [-1], [rows - 20]], device="cuda", dtype=torch.int32)
    quantize_fp4(x, q, scales, slots=slots)
    alone = torch.empty(5, k // 2, device="cuda", dtype=torch.uint8), torch.empty(5, k // 32, device="cuda", dtype=torch.uint8)
    quantize_fp4(x, *alone)
    at = slots[slots >= 0].long()
    assert torch.equal(q[at], alone[0][(slots >= 0).squeeze(1)])
    assert torch.equal(scales[at], alone[1][(slots >= 0).squeeze(1)])
    out = torch.empty(rows, k, device="cuda", dtype=BF16)
    dequantize_fp4(q, scales, out)
    assert torch.equal(out[at].double(), values(q[at], scales[at]))


@pytest.mark.parametrize("rows, n", [(36000, 60000), (60001, 36001)])
def test_results_behind_2_31_elements(rows, n):
    k = 64
    a, a_scales = operand((rows, k), 1)
    b, b_scales = operand((n, k), 2, 115, 126)
    out = torch.empty(rows, n, device="cuda", dtype=BF16)
    gemm_fp4(a, a_scales, b, b_scales, out)
    for lo in (0, rows - 300):
        ref, magnitude = product(values(a[lo:lo + 300], a_scales[lo:lo + 300]), values(b, b_scales).unsqueeze(0), [(0, 300)])
        check(out[lo:lo + 300], ref, magnitude, k)


def test_weights_behind_2_31_bytes():
    experts, n, k = 20, 16384, 16384  # 2.7 GB of codes
    b = torch.randint(0, 256, (experts, n, k // 2), device="cuda", dtype=torch.uint8)
    b_scales = torch.randint(115, 120, (experts, n, k // 32), device="cuda", dtype=torch.uint8)
    counts = [0] * (experts - 2) + [5, 40]
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), device="cuda", dtype=torch.int32)
    a, a_scales = operand((45, k), 1)
    out = torch.empty(45, n, device="cuda", dtype=BF16)
    gemm_fp4(a, a_scales, b, b_scales, out, offsets=offsets)
    for e, lo, hi in ((experts - 2, 0, 5), (experts - 1, 5, 45)):
        ref, magnitude = product(values(a[lo:hi], a_scales[lo:hi]), values(b[e], b_scales[e]).unsqueeze(0), [(0, hi - lo)])
        check(out[lo:hi], ref, magnitude, k)


def test_sort_of_many_choices():
    """Millions of choices, so that a warp's part takes many rounds, over the most experts there can be."""
    ids = torch.randint(-1, 1025, (700001, 7), device="cuda")
    offsets = torch.empty(1025, device="cuda", dtype=torch.int32)
    slots = torch.empty(ids.shape, device="cuda", dtype=torch.int32)
    expert_sort(ids, offsets, slots)
    flat = ids.reshape(-1)
    here = (flat >= 0) & (flat < 1024)
    order = torch.sort(flat[here], stable=True).indices
    want = torch.full_like(flat, -1)
    want[here.nonzero().squeeze(1)[order]] = torch.arange(order.numel(), device="cuda")
    assert torch.equal(slots.reshape(-1).long(), want)
    assert torch.equal(offsets[1:].long(), torch.bincount(flat[here], minlength=1024).cumsum(0)) and offsets[0] == 0


def test_rows_as_wide_as_they_come():
    """One token whose row is shared among many CTAs, and more choices than a warp has lanes."""
    width = 3 * 2 ** 20 + 8
    x, w = _randn((1, width), 1), _randn((1, 40), 2, torch.float32)
    slots = torch.arange(40, device="cuda", dtype=torch.int32).view(1, 40).flip(1).contiguous()
    rows = torch.zeros(40, width, device="cuda", dtype=BF16)
    expert_dispatch(x, slots, rows, weights=w)
    ref = x.double() * w.double().flip(1).view(40, 1)
    assert ((rows.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -23) * ref.abs() + 2.0 ** -133).all()
    out = torch.empty_like(x)
    expert_combine(rows, slots, out)
    total, magnitude = rows.double().sum(0), rows.double().abs().sum(0)
    assert ((out[0].double() - total).abs() <= 2.0 ** -8 * total.abs() + 42 * 2.0 ** -23 * magnitude + 2.0 ** -133).all()


@pytest.mark.parametrize("dtype, width", [(BF16, 2 ** 30 + 9), (torch.float32, 2 ** 29 + 9), (BF16, 2 ** 30 + 8)])
def test_rows_behind_2_31_bytes_in_one(dtype, width):
    """Rows of more than 2^31 bytes each, one of them the matrix's first and one its last."""
    y = torch.zeros(2, width, device="cuda", dtype=dtype)
    places = torch.tensor([0, 1, 255, 256, width // 2, width // 2 + 1, width - 9, width - 2, width - 1], device="cuda")
    some = _randn((2, places.numel()), 3, dtype)
    y[:, places] = some
    slots, w = torch.tensor([[1, 0]], device="cuda", dtype=torch.int32), torch.tensor([[0.5, 2.0]], device="cuda")
    out = torch.full((1, width), float("nan"), device="cuda", dtype=dtype)
    expert_combine(y, slots, out, weights=w)
    want = (0.5 * some[1].float() + 2.0 * some[0].float()).to(dtype)  # powers of two: one rounding of fp32 sums each way
    assert torch.equal(out[0, places], want)
    assert int(torch.count_nonzero(out)) == int(torch.count_nonzero(want))
    grad_w = torch.empty_like(w)
    del want
    expert_combine_grad(out, y, slots, w, y, grad_w)  # over y: at most nine products that are not 0
    ref = (out[0, places].double() * some.double()).sum(1).flip(0)
    size = (out[0, places].double() * some.double()).abs().sum(1).flip(0)
    assert ((grad_w[0].double() - ref).abs() <= 18 * 2.0 ** -24 * size).all()
    assert torch.equal(y[1, places], (0.5 * out[0, places].float()).to(dtype)) and torch.equal(y[0, places], 2 * out[0, places])
    expert_dispatch(out, slots, y)
    assert torch.equal(y[0, places], out[0, places]) and torch.equal(y[1, places], out[0, places])
    assert int(torch.count_nonzero(y)) == 2 * int(torch.count_nonzero(out))


@pytest.mark.parametrize("k", [2 ** 20, 2 ** 20 + 32])
def test_product_of_a_long_k(k):
    a, a_scales = operand((3, k), 1, 120, 124)
    b, b_scales = operand((5, k), 2, 110, 114)
    out = torch.empty(3, 5, device="cuda", dtype=BF16)
    gemm_fp4(a, a_scales, b, b_scales, out)
    check(out, *product(values(a, a_scales), values(b, b_scales).unsqueeze(0), [(0, 3)]), k)
