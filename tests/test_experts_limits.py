"""Sizes at the end of 32 bits: the expert-layer products refuse them before a launch.

The kernels count rows and columns in 32-bit integers, rounded up to whole tiles and stepped past the end by a stage.
Close to 2^31 such a count wraps: a loop over stages would not end, and a tile count would be negative.
"""
from __future__ import annotations

import pytest

from teamredbench_b200 import _native

P = 4096  # an aligned address that is never read: every call below is refused first
BF16 = 1
LARGEST = 2130706432
INT_MAX = 2 ** 31 - 1


def _wraps(x):
    return (x + 2 ** 31) % 2 ** 32 - 2 ** 31


@pytest.mark.parametrize("rows", [LARGEST, LARGEST - 255, LARGEST // 2 + 1])
def test_counts_up_to_the_largest_size_stay_in_32_bits(rows):
    chunks = _wraps(rows + 255) // 256  # of a group, in the products
    assert 0 < chunks and 0 < _wraps(rows + chunks - 1) and 0 < _wraps(rows + 2 * 256)
    last_stage = (rows - 1) // 128 * 128  # of a group, in the gradient
    assert _wraps(last_stage + 128) >= rows


def test_the_counts_would_wrap_just_above():
    assert _wraps((INT_MAX - 1) // 128 * 128 + 128) < 0
    assert _wraps(INT_MAX + 255) < 0


@pytest.mark.parametrize("rows, n, k", [(INT_MAX, 8, 8), (LARGEST + 1, 8, 8), (8, INT_MAX - 7, 8), (8, 8, INT_MAX - 7),
                                        (8, LARGEST + 8, 8)])
def test_grouped_entries_refuse(rows, n, k):
    lib = _native.load()
    for status in (lib.trb_grouped_gemm_launch(BF16, 1, rows, n, k, P, P, 0, P, P, None),
                   lib.trb_grouped_wgrad_launch(BF16, 1, rows, n, k, P, P, P, P, None)):
        assert status == 1
        assert f"at most {LARGEST}" in _native.last_error()


@pytest.mark.parametrize("rows, n", [(INT_MAX, 8), (8, INT_MAX), (LARGEST + 1, 8)])
def test_gemv_w4_entry_refuses(rows, n):
    assert _native.load().trb_gemv_w4_launch(BF16, 1, rows, n, 64, 32, P, P, P, None, None, P, None) == 1
    assert f"at most {LARGEST}" in _native.last_error()


@pytest.mark.parametrize("launch", [
    lambda r, n, k: _native.grouped_gemm_launch("bfloat16", 1, r, n, k, P, P, "row_major", P, P),
    lambda r, n, k: _native.grouped_wgrad_launch("bfloat16", 1, r, n, k, P, P, P, P),
    lambda r, n, k: _native.gemv_w4_launch("bfloat16", 1, r, n, k, 32, P, P, P, None, None, P),
], ids=["grouped_gemm", "grouped_wgrad", "gemv_w4"])
@pytest.mark.parametrize("which", "rnk")
def test_sizes_past_32_bits_are_not_cut(launch, which):
    """Cut to 32 bits, 2^32 rows would be a call of no rows, done at once, and n or k those of a smaller matrix."""
    size = {"r": 0, "n": 64, "k": 64}
    size[which] += 2 ** 32
    with pytest.raises(ValueError, match="32 bits"):
        launch(size["r"], size["n"], size["k"])
