"""GPU tests of the products grouped by expert (grouped_gemm, grouped_gemm_wgrad) against plain 64-bit forms,
with elementwise bounds derived from the number formats (tests/grouped_helpers.py)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import grouped_gemm, grouped_gemm_wgrad  # noqa: E402
from tests.grouped_helpers import DTYPES, bounds, check, offsets_of, product, randn, wgrad  # noqa: E402

NAN = float("nan")

# rows per group: one row; exact tiles and one more or less; empty groups first, last and between; many groups
COUNTS = {
    "one_row": [1],
    "one_row_of_many": [0, 0, 1, 0],
    "edges": [31, 32, 33, 0, 255, 256, 257],
    "chunks": [513, 0, 769, 96, 1],
    "many": [(7 * i * i) % 41 for i in range(97)],
    "none": [0, 0, 0],
}
# (k, n): one 8-wide sliver, below / at / above the 64-wide k-block and the 128- and 256-wide tiles
WIDTHS = [(8, 8), (64, 128), (72, 264), (200, 136), (1032, 520)]


@pytest.fixture(autouse=True)
def no_device_error():
    assert _native.device_error(0, clear=True) == 0
    yield
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0


def _weights(groups, k, n, dtype, seed, b_transposed):
    return randn((groups, n, k) if b_transposed else (groups, k, n), dtype, seed, k ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b_transposed", [False, True])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("k, n", WIDTHS)
def test_product(dtype, b_transposed, counts, k, n):
    counts = COUNTS[counts]
    rows = sum(counts)
    offsets = offsets_of(counts)
    a = randn((rows, k), dtype, 1)
    b = _weights(len(counts), k, n, dtype, 2, b_transposed)
    out = torch.full((rows, n), NAN, device="cuda", dtype=DTYPES[dtype])
    assert grouped_gemm(a, b, offsets, out, b_transposed=b_transposed) is out
    check(dtype, out, *product(a, b, offsets, b_transposed), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("k, n", WIDTHS)
def test_wgrad(dtype, counts, k, n):
    counts = COUNTS[counts]
    rows = sum(counts)
    offsets = offsets_of(counts)
    a, grad = randn((rows, k), dtype, 3), randn((rows, n), dtype, 4)
    out = torch.full((len(counts), k, n), NAN, device="cuda", dtype=DTYPES[dtype])
    assert grouped_gemm_wgrad(a, grad, offsets, out) is out
    check(dtype, out, *wgrad(a, grad, offsets), max(counts))
    for e, c in enumerate(counts):
        if c == 0:
            assert not out[e].any()


@pytest.mark.parametrize("left", range(1, 17))
def test_wgrad_takes_nothing_of_the_rows_behind(left):
    """Rows behind a group's last one, in its 16-row step and its 64-row stage, hold infinities and NaN."""
    counts = [64 + left, 48, left]
    gap = 70
    rows = sum(counts) + gap
    offsets = offsets_of(counts)
    a, grad = randn((rows, 136), "bfloat16", 5), randn((rows, 264), "bfloat16", 6)
    ref = wgrad(a, grad, offsets)
    poisoned = torch.empty((3, 136, 264), device="cuda", dtype=torch.bfloat16)
    a[sum(counts):], grad[sum(counts):] = float("inf"), NAN
    grouped_gemm_wgrad(a, grad, offsets, poisoned)
    check("bfloat16", poisoned, *ref, max(counts))
    # the same between groups: the middle group's rows are not numbers, the other gradients do not change
    a[64 + left:112 + left], grad[64 + left:112 + left] = NAN, float("-inf")
    again = torch.empty_like(poisoned)
    grouped_gemm_wgrad(a, grad, offsets, again)
    assert torch.equal(again[0], poisoned[0]) and torch.equal(again[2], poisoned[2])
    assert torch.isnan(again[1]).all()


@pytest.mark.parametrize("b_transposed", [False, True])
def test_product_keeps_rows_and_groups_apart(b_transposed):
    """NaN in the weights of groups without rows, in rows outside every group and in single rows stay there;
    rows outside every group keep what out held."""
    counts = [40, 0, 33, 0, 1]
    first, k, n = 11, 104, 200
    rows = first + sum(counts) + 9
    offsets = offsets_of(counts, first)
    a = randn((rows, k), "float16", 7)
    b = _weights(5, k, n, "float16", 8, b_transposed)
    ref, mag = product(a, b, offsets, b_transposed)
    a[:first], a[rows - 9:] = NAN, float("inf")
    a[20], a[55, 3] = NAN, float("inf")
    b[1], b[3] = NAN, float("inf")
    out = torch.full((rows, n), 7.0, device="cuda", dtype=torch.float16)
    grouped_gemm(a, b, offsets, out, b_transposed=b_transposed)
    assert torch.all(out[:first] == 7.0) and torch.all(out[rows - 9:] == 7.0)
    assert torch.isnan(out[20]).all()
    assert not torch.isfinite(out[55]).any()
    keep = torch.ones(rows, dtype=torch.bool)
    keep[:first] = keep[rows - 9:] = keep[20] = keep[55] = False
    keep = keep.cuda()
    check("float16", out[keep], ref[keep], mag[keep], k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_by_differences(dtype):
    """With whole numbers small enough that every sum is exact in 16 bits, L(a, b) = sum(c * out) changes by exactly
    <gradient, step> when a or b takes a step; the gradients are the operators' own."""
    counts, k, n = [5, 0, 37, 18], 40, 72
    rows, offsets = sum(counts), offsets_of(counts)
    g = torch.Generator(device="cuda").manual_seed(9)

    def whole(shape, low, high, keep):
        x = torch.randint(low, high + 1, shape, generator=g, device="cuda")
        return (x * (torch.rand(shape, generator=g, device="cuda") < keep)).to(DTYPES[dtype])

    a, da = whole((rows, k), -2, 2, 0.5), whole((rows, k), -1, 1, 0.2)
    b, db = whole((4, k, n), -2, 2, 0.5), whole((4, k, n), -1, 1, 0.2)
    c = whole((rows, n), -1, 1, 0.3)

    def loss(x, w):
        out = torch.empty((rows, n), device="cuda", dtype=DTYPES[dtype])
        grouped_gemm(x, w, offsets, out)
        assert out.abs().max() < 256
        return (c.double() * out.double()).sum().item()

    grad_a = torch.empty_like(a)
    grouped_gemm(c, b, offsets, grad_a, b_transposed=True)
    grad_b = torch.empty_like(b)
    grouped_gemm_wgrad(a, c, offsets, grad_b)
    assert grad_a.abs().max() < 256 and grad_b.abs().max() < 256
    assert loss(a + da, b) - loss(a, b) == (grad_a.double() * da.double()).sum().item()
    assert loss(a, b + db) - loss(a, b) == (grad_b.double() * db.double()).sum().item()
    # weights kept (groups, n, k): the gradient with the operands exchanged is the transpose
    grad_bt = torch.empty((4, n, k), device="cuda", dtype=DTYPES[dtype])
    grouped_gemm_wgrad(c, a, offsets, grad_bt)
    assert torch.equal(grad_bt, grad_b.transpose(1, 2))


def test_same_bits_every_time_and_on_another_stream():
    counts, k, n = [100, 0, 300, 28, 600], 520, 776
    rows, offsets = sum(counts), offsets_of(counts)
    a, b, grad = randn((rows, k), "bfloat16", 10), randn((5, k, n), "bfloat16", 11), randn((rows, n), "bfloat16", 12)
    first = grouped_gemm(a, b, offsets, torch.empty((rows, n), device="cuda", dtype=torch.bfloat16))
    first_w = grouped_gemm_wgrad(a, grad, offsets, torch.empty((5, k, n), device="cuda", dtype=torch.bfloat16))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for use_context in (True, False):
        out, out_w = torch.zeros_like(first), torch.zeros_like(first_w)
        torch.cuda.synchronize()
        if use_context:
            with torch.cuda.stream(side):
                grouped_gemm(a, b, offsets, out)
                grouped_gemm_wgrad(a, grad, offsets, out_w)
        else:
            grouped_gemm(a, b, offsets, out, stream=side)
            grouped_gemm_wgrad(a, grad, offsets, out_w, stream=side)
        side.synchronize()
        assert torch.equal(out, first) and torch.equal(out_w, first_w)


def test_operands_of_the_previous_launch():
    """Chained calls: each reads what the one before has just written, offsets among it."""
    counts, d = [130, 7, 0, 250], 384
    rows = sum(counts)
    want = offsets_of(counts)
    a, b = randn((rows, d), "bfloat16", 13), randn((4, d, d), "bfloat16", 14, d ** -0.5)
    x, y = a.clone(), torch.empty_like(a)
    for _ in range(8):
        offsets = torch.zeros(5, dtype=torch.int32, device="cuda")
        offsets.copy_(want)
        grouped_gemm(x, b, offsets, y)
        x, y = y, x
    ref = a
    for _ in range(8):
        ref = product(ref, b, want, False)[0].to(torch.bfloat16)
    torch.cuda.synchronize()
    # eight roundings apart at most where fp32 and fp64 sums round to different neighbours
    assert (x.double() - ref.double()).norm() <= 8 * 2.0 ** -8 * ref.double().norm()


def test_captured_in_a_graph_with_new_offsets():
    counts, k, n = [64, 64, 64], 128, 256
    offsets = offsets_of(counts)
    a, b = randn((192, k), "float16", 15), randn((3, k, n), "float16", 16, k ** -0.5)
    out = torch.empty((192, n), device="cuda", dtype=torch.float16)
    grouped_gemm(a, b, offsets, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grouped_gemm(a, b, offsets, out)
    for other in ([64, 64, 64], [0, 191, 1], [192, 0, 0]):
        offsets.copy_(offsets_of(other))
        out.zero_()
        graph.replay()
        check("float16", out, *product(a, b, offsets, False), k)


def test_results_past_32_bit_offsets():
    k, n, rows = 64, 16384, 140000  # 2.3e9 results
    offsets = offsets_of([70001, 69999])
    a, b = randn((rows, k), "bfloat16", 17), randn((2, k, n), "bfloat16", 18, k ** -0.5)
    out = torch.empty((rows, n), device="cuda", dtype=torch.bfloat16)
    grouped_gemm(a, b, offsets, out)
    for lo in (0, 69990, rows - 300):
        part = slice(lo, lo + 300)
        local = (offsets - lo).clamp(0, 300).to(torch.int32)
        check("bfloat16", out[part], *product(a[part], b, local, False), k)


def test_gradients_past_32_bit_offsets():
    groups, k, n = 40, 8192, 8192  # 2.7e9 results
    counts = [3] * groups
    offsets = offsets_of(counts)
    a, grad = randn((3 * groups, k), "bfloat16", 19), randn((3 * groups, n), "bfloat16", 20)
    out = torch.empty((groups, k, n), device="cuda", dtype=torch.bfloat16)
    grouped_gemm_wgrad(a, grad, offsets, out)
    for e in (0, 31, groups - 1):
        lo, hi = bounds(offsets)[e]
        check("bfloat16", out[e:e + 1], *wgrad(a[lo:hi], grad[lo:hi], offsets_of([hi - lo])), 3)


@pytest.mark.parametrize("bad", [[0, 5, 4, 8], [-1, 2, 4, 8], [0, 2, 4, 9], [0, 2 ** 31 - 1, 4, 8], [8, 0, 8, 0]])
def test_wrong_offsets_compute_nothing_and_set_the_error_word(bad):
    offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
    a, b = randn((8, 64), "bfloat16", 21), randn((3, 64, 64), "bfloat16", 22)
    out = torch.full((8, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    grouped_gemm(a, b, offsets, out)
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 7
    assert torch.all(out == 3.0)
    dw = torch.full((3, 64, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    grouped_gemm_wgrad(a, a, offsets, dw)
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 7
    assert torch.all(dw == 3.0)


def test_refusals():
    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, device="cuda", dtype=dtype)

    offsets = offsets_of([4, 4])
    a, b, out = t(8, 64), t(2, 64, 32), t(8, 32)
    with pytest.raises(ValueError, match="incompatible shapes"):
        grouped_gemm(a, b, offsets, out, b_transposed=True)
    with pytest.raises(ValueError, match="out must be"):
        grouped_gemm(a, b, offsets, t(8, 64))
    with pytest.raises(ValueError, match="2-D a and a 3-D b"):
        grouped_gemm(a, b[0], offsets, out)
    with pytest.raises(ValueError, match="one dtype"):
        grouped_gemm(a, b.half(), offsets, out)
    with pytest.raises(ValueError, match="offsets must be 3 int32"):
        grouped_gemm(a, b, offsets.long(), out)
    with pytest.raises(ValueError, match="offsets must be 3 int32"):
        grouped_gemm(a, b, offsets[:2], out)
    with pytest.raises(ValueError, match="CUDA device"):
        grouped_gemm(a, b, offsets.cpu(), out)
    with pytest.raises(ValueError, match="contiguous"):
        grouped_gemm(t(64, 8).T, b, offsets, out)
    with pytest.raises(_native.NativeError, match="multiples of 8"):
        grouped_gemm(t(8, 60), t(2, 60, 32), offsets, out)
    with pytest.raises(_native.NativeError, match="16-byte aligned"):
        grouped_gemm(t(8 * 64 + 1)[1:].view(8, 64), b, offsets, out)
    with pytest.raises(_native.NativeSkipped, match="unsupported dtype"):
        grouped_gemm(a.float(), b.float(), offsets, out.float())
    with pytest.raises(_native.NativeSkipped, match="at most 1024 groups"):
        grouped_gemm(a, t(1025, 64, 32), t(1026, dtype=torch.int32), out)
    with pytest.raises(ValueError, match="same number of rows"):
        grouped_gemm_wgrad(a, t(7, 32), offsets, t(2, 64, 32))
    with pytest.raises(ValueError, match="out must be"):
        grouped_gemm_wgrad(a, t(8, 32), offsets, t(2, 32, 64))
    with pytest.raises(_native.NativeError, match="multiples of 8"):
        grouped_gemm_wgrad(a, t(8, 36), offsets, t(2, 64, 36))
