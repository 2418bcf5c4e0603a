"""The expert-layer products at the sizes that reach each of their variants: K split over clusters of every size for
both tile heights, column tiles of a gradient in a last run of fewer than eight, and the 4-bit product's scales and
zero points read as vectors or one at a time.  Bounds as in tests/grouped_helpers.py."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import gemv_w4, grouped_gemm, grouped_gemm_wgrad  # noqa: E402
from tests.grouped_helpers import DTYPES, check, offsets_of, product, randn, w4_operands, w4_weights, wgrad  # noqa: E402

NAN = float("nan")


@pytest.fixture(autouse=True)
def no_device_error():
    assert _native.device_error(0, clear=True) == 0
    yield
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0


def _product(dtype, counts, k, n, b_transposed, seed):
    rows, offsets = sum(counts), offsets_of(counts)
    a = randn((rows, k), dtype, seed)
    b = randn((len(counts), n, k) if b_transposed else (len(counts), k, n), dtype, seed + 1, k ** -0.5)
    out = torch.full((rows, n), NAN, device="cuda", dtype=DTYPES[dtype])
    grouped_gemm(a, b, offsets, out, b_transposed=b_transposed)
    check(dtype, out, *product(a, b, offsets, b_transposed), k)


# 4, 9, 17 and 40 k-blocks of 64 (the last one partial) allow clusters of 2, 4, 8 and 8; up to 4 rows a group on
# average take tiles of 16 rows, more take 64.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b_transposed", [False, True])
@pytest.mark.parametrize("k", [8, 200, 520, 1032, 2504])
@pytest.mark.parametrize("counts", [[2, 0, 1], [17, 0, 0, 0, 1], [65, 64, 1], [90]])
def test_split_over_clusters(dtype, b_transposed, k, counts):
    _product(dtype, counts, k, 264, b_transposed, k + len(counts))


# One group of 50 rows is one tile of 64 rows for each 128 columns and one place more, so n = 128 t gives 1 t tiles
# at work; around the counts at which the clusters of 8, 4 and 2 that the GPU holds at once are full or just overrun.
@pytest.mark.parametrize("tiles", [15, 16, 18, 19, 33, 34, 37, 38, 74, 75])
@pytest.mark.parametrize("counts", [[50], [3]])
@pytest.mark.parametrize("b_transposed", [False, True])
def test_split_around_full_clusters(tiles, counts, b_transposed):
    _product("bfloat16", counts, 1096, 128 * tiles, b_transposed, tiles)


# 9 and 11 column tiles: a last run of 1 and of 3, partial last tiles both ways.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2056, 2304, 2568])
@pytest.mark.parametrize("k", [256, 520])
def test_gradient_with_a_partial_run_of_column_tiles(dtype, n, k):
    counts = [130, 0, 33, 5]
    offsets = offsets_of(counts)
    a, grad = randn((168, k), dtype, n), randn((168, n), dtype, k)
    out = torch.full((4, k, n), NAN, device="cuda", dtype=DTYPES[dtype])
    grouped_gemm_wgrad(a, grad, offsets, out)
    check(dtype, out, *wgrad(a, grad, offsets), max(counts))
    assert not out[1].any()


def _shifted(t, by):
    """The same values `by` elements behind an aligned address."""
    room = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)[by:by + t.numel()]
    return room.copy_(t.flatten()).view(t.shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group, k", [(32, 128), (32, 512), (32, 640), (32, 4096), (64, 128), (64, 1152), (128, 1024)])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("shift_scales, shift_zeros", [(0, 0), (1, 0), (2, 2), (0, 1), (3, 3), (4, 4)])
def test_scales_and_zero_points_at_any_element(dtype, group, k, with_zeros, shift_scales, shift_zeros):
    """k of whole vectors of scales, the scales and zero points at every alignment of such a vector."""
    n, rows = 77, 11
    q, scales, zeros = w4_operands(1, n, k, group, dtype, k + group, with_zeros)
    x = randn((rows, k), dtype, 3)
    out = torch.full((rows, n), NAN, device="cuda", dtype=DTYPES[dtype])
    gemv_w4(x, q[0], _shifted(scales[0], shift_scales), out,
            zeros=_shifted(zeros[0], shift_zeros) if with_zeros else None)
    check(dtype, out, *product(x, w4_weights(q, scales, zeros), offsets_of([rows]), True), k)


# Rows of x that fit in shared memory at once: 16 up to k = 4096, then 10, 9, 8, 4, 2; the rows come in as many passes.
@pytest.mark.parametrize("k", [4096, 6144, 7168, 8192, 14336, 28672])
@pytest.mark.parametrize("rows", [8, 9, 16, 21])
def test_rows_in_several_passes(k, rows):
    q, scales, zeros = w4_operands(1, 33, k, 128, "bfloat16", k, True)
    x = randn((rows, k), "bfloat16", 4)
    out = torch.full((rows, 33), NAN, device="cuda", dtype=torch.bfloat16)
    gemv_w4(x, q[0], scales[0], out, zeros=zeros[0])
    check("bfloat16", out, *product(x, w4_weights(q, scales, zeros), offsets_of([rows]), True), k)
