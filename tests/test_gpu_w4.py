"""GPU tests of gemv_w4 (few rows times 4-bit weights with group scales) against the 64-bit form, with elementwise
bounds derived from the number formats (tests/grouped_helpers.py)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import gemv_w4  # noqa: E402
from tests.grouped_helpers import DTYPES, check, offsets_of, product, randn, w4_operands, w4_weights  # noqa: E402

NAN = float("nan")


@pytest.fixture(autouse=True)
def no_device_error():
    assert _native.device_error(0, clear=True) == 0
    yield
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0


def _run(dtype, rows, n, k, group, with_zeros, counts=None, seed=1):
    groups = 1 if counts is None else len(counts)
    q, scales, zeros = w4_operands(groups, n, k, group, dtype, seed, with_zeros)
    x = randn((rows, k), dtype, seed + 2)
    offsets = offsets_of([rows] if counts is None else counts)
    out = torch.full((rows, n), NAN, device="cuda", dtype=DTYPES[dtype])
    if counts is None:
        got = gemv_w4(x, q[0], scales[0], out, zeros=None if zeros is None else zeros[0])
    else:
        got = gemv_w4(x, q, scales, out, zeros=zeros, offsets=offsets)
    assert got is out
    check(dtype, out, *product(x, w4_weights(q, scales, zeros), offsets, True), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 15, 16, 17, 40])
@pytest.mark.parametrize("group, k", [(32, 1056), (64, 512), (128, 4096), (256, 768), (2048, 2048)])
def test_rows_and_groups(dtype, rows, group, k):
    _run(dtype, rows, 200, k, group, with_zeros=rows % 2 == 1)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 127, 128, 129, 1001])
@pytest.mark.parametrize("group, k", [(32, 32), (32, 64), (32, 288), (64, 192), (128, 1152), (128, 128), (512, 5120)])
@pytest.mark.parametrize("rows", [1, 11])
def test_widths(n, group, k, rows):
    _run("bfloat16", rows, n, k, group, with_zeros=True, seed=n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[1], [0, 1, 0, 0, 2], [3, 0, 8, 9, 1, 0, 17], [1] * 70, [0, 0], [40, 1, 30]])
@pytest.mark.parametrize("group, k, n", [(128, 1024, 272), (32, 416, 75)])
def test_experts(dtype, counts, group, k, n):
    _run(dtype, sum(counts), n, k, group, with_zeros=True, counts=counts)


@pytest.mark.parametrize("rows", [1, 8, 16])
def test_long_k(rows):
    _run("bfloat16", rows, 48, 65536, 128, with_zeros=False)


@pytest.mark.parametrize("rows", [1, 16])
def test_many_tiles_for_each_block(rows):
    _run("float16", rows, 20011, 1024, 64, with_zeros=True)


def test_every_weight_and_zero_point():
    """Unit rows pick single weights: all 16 values of q against all 16 zero points come out exactly."""
    k, n = 32, 256
    q = torch.arange(16, device="cuda").repeat(16)  # output i: q = i % 16, zero point i // 16
    packed = (q | q << 4).to(torch.uint8)[:, None].expand(n, k // 2).contiguous()
    zeros = torch.arange(16, device="cuda").repeat_interleave(16).to(torch.uint8)[:, None].contiguous()
    for dtype in DTYPES.values():
        x = torch.eye(k, device="cuda", dtype=dtype)
        scales = torch.full((n, 1), 0.5, device="cuda", dtype=dtype)
        out = torch.empty((k, n), device="cuda", dtype=dtype)
        gemv_w4(x, packed, scales, out, zeros=zeros)
        want = 0.5 * (q - zeros[:, 0].long()).double()
        assert torch.equal(out.double(), want.expand(k, n))


def test_order_of_the_weights():
    """Unit rows against weights that differ along k: place j of a row is the low, then the high half of byte j // 2."""
    k, n = 512, 40
    q, scales, _ = w4_operands(1, n, k, 32, "bfloat16", 3, False)
    x = torch.eye(k, device="cuda", dtype=torch.bfloat16)
    out = torch.empty((k, n), device="cuda", dtype=torch.bfloat16)
    gemv_w4(x, q[0], scales[0], out)
    assert torch.equal(out, w4_weights(q, scales, None)[0].T.to(torch.bfloat16))


def test_infinities_and_nan_stay_in_their_rows():
    k, n = 256, 64
    q, scales, _ = w4_operands(1, n, k, 64, "bfloat16", 4, False)
    x = randn((6, k), "bfloat16", 5)
    ref = product(x, w4_weights(q, scales, None), offsets_of([6]), True)
    x[1, 9], x[4, 200] = NAN, float("inf")
    out = torch.empty((6, n), device="cuda", dtype=torch.bfloat16)
    gemv_w4(x, q[0], scales[0], out)
    assert torch.isnan(out[1]).all()
    w = w4_weights(q, scales, None)[0][:, 200]
    assert torch.isnan(out[4][w == 0]).all()
    assert torch.equal(out[4][w != 0], torch.where(w[w != 0] > 0, float("inf"), -float("inf")).to(torch.bfloat16))
    keep = [0, 2, 3, 5]
    check("bfloat16", out[keep], ref[0][keep], ref[1][keep], k)


def test_rows_outside_every_group_keep_their_values():
    counts, first, k, n = [2, 0, 1], 3, 128, 50
    q, scales, zeros = w4_operands(3, n, k, 32, "float16", 6, True)
    offsets = offsets_of(counts, first)
    x = randn((9, k), "float16", 7)
    x[:3] = NAN
    scales[1] = NAN  # of a group without rows
    out = torch.full((9, n), 5.0, device="cuda", dtype=torch.float16)
    gemv_w4(x, q, scales, out, zeros=zeros, offsets=offsets)
    assert torch.all(out[:3] == 5.0) and torch.all(out[6:] == 5.0)
    ref, mag = product(x, w4_weights(q, scales, zeros), offsets, True)
    check("float16", out[3:6], ref[3:6], mag[3:6], k)


def test_same_bits_every_time_and_on_another_stream():
    q, scales, zeros = w4_operands(1, 3000, 4096, 128, "bfloat16", 8, True)
    x = randn((5, 4096), "bfloat16", 9)
    first = gemv_w4(x, q[0], scales[0], torch.empty((5, 3000), device="cuda", dtype=torch.bfloat16), zeros=zeros[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        out = torch.zeros_like(first)
        torch.cuda.synchronize()
        gemv_w4(x, q[0], scales[0], out, zeros=zeros[0], stream=side)
        side.synchronize()
        assert torch.equal(out, first)


def test_weights_past_32_bit_offsets():
    groups, n, k = 3, 40000, 65536  # 3.9e9 bytes of q
    counts = [1, 0, 2]
    q = torch.randint(0, 256, (groups, n, k // 2), device="cuda", dtype=torch.uint8)
    scales = randn((groups, n, k // 1024), "bfloat16", 10, 0.05)
    x = randn((3, k), "bfloat16", 11)
    out = torch.full((3, n), NAN, device="cuda", dtype=torch.bfloat16)
    gemv_w4(x, q, scales, out, offsets=offsets_of(counts))
    for part in (slice(0, 100), slice(n - 100, n)):
        w = w4_weights(q[:, part], scales[:, part], None)
        check("bfloat16", out[:, part], *product(x, w, offsets_of(counts), True), k)


@pytest.mark.parametrize("bad", [[0, 5, 4, 8], [-1, 2, 4, 8], [0, 2, 4, 9]])
def test_wrong_offsets_compute_nothing_and_set_the_error_word(bad):
    q, scales, _ = w4_operands(3, 64, 128, 32, "bfloat16", 12, False)
    x = randn((8, 128), "bfloat16", 13)
    out = torch.full((8, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    gemv_w4(x, q, scales, out, offsets=torch.tensor(bad, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 7
    assert torch.all(out == 3.0)


def test_refusals():
    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, device="cuda", dtype=dtype)

    x, q, s, out = t(2, 128), t(10, 64, dtype=torch.uint8), t(10, 4), t(2, 10)
    gemv_w4(x, q, s, out)
    gemv_w4(t(0, 128), q, s, t(0, 10))  # no rows: nothing to do
    with pytest.raises(ValueError, match="128 weights a row for k = 64"):
        gemv_w4(t(2, 64), q, s, out)
    with pytest.raises(ValueError, match="scales must be"):
        gemv_w4(x, q, t(10, 3), out)
    with pytest.raises(ValueError, match="scales must be"):
        gemv_w4(x, q, t(9, 4), out)
    with pytest.raises(ValueError, match="zeros must be"):
        gemv_w4(x, q, s, out, zeros=t(10, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="out must be"):
        gemv_w4(x, q, s, t(2, 11))
    with pytest.raises(ValueError, match="one dtype"):
        gemv_w4(x, q, s.half(), out)
    with pytest.raises(ValueError, match="must be uint8"):
        gemv_w4(x, q.to(torch.int8), s, out)
    with pytest.raises(ValueError, match="2 groups need offsets"):
        gemv_w4(x, t(2, 10, 64, dtype=torch.uint8), t(2, 10, 4), out)
    with pytest.raises(ValueError, match="contiguous"):
        gemv_w4(x, t(64, 10, dtype=torch.uint8).T, s, out)
    with pytest.raises(_native.NativeSkipped, match="group size"):
        gemv_w4(x, q, t(10, 8), out)  # groups of 16
    with pytest.raises(_native.NativeSkipped, match="group size"):
        gemv_w4(t(2, 96), t(10, 48, dtype=torch.uint8), t(10, 1), out)  # a group of 96
    with pytest.raises(_native.NativeSkipped, match="unsupported dtype"):
        gemv_w4(x.float(), q, s.float(), out.float())
    with pytest.raises(_native.NativeSkipped, match="at most 65536"):
        gemv_w4(t(1, 131072), t(1, 65536, dtype=torch.uint8), t(1, 1024), t(1, 1))
    with pytest.raises(_native.NativeError, match="16-byte aligned"):
        gemv_w4(t(2 * 128 + 1)[1:].view(2, 128), q, s, out)
