"""GPU tests of microscaled 4-bit floating point (quantize_fp4, dequantize_fp4, gemm_fp4) against plain 64-bit forms:
codes and scales are equal, products stay within bounds derived from the number formats (tests/fp4_helpers.py)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import (  # noqa: E402
    dequantize_fp4, expert_combine, expert_sort, gemm_fp4, quantize_fp4)
from tests.fp4_helpers import DTYPES, check, operand, packed, pitch, product, quantised, values  # noqa: E402
from tests.grouped_helpers import bounds, offsets_of  # noqa: E402

NAN = float("nan")


@pytest.fixture(autouse=True)
def no_device_error():
    assert _native.device_error(0, clear=True) == 0
    yield
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0


def _randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _quantize(x):
    rows, k = x.shape
    q = torch.full((rows, k // 2), 0x55, device="cuda", dtype=torch.uint8)
    scales = torch.full((rows, pitch(k)), 0x55, device="cuda", dtype=torch.uint8)
    assert quantize_fp4(x, q, scales) == (q, scales)
    return q, scales


def _same(x, q, scales):
    codes, exponents = quantised(x)
    blocks = x.shape[1] // 32
    assert torch.equal(scales[:, :blocks].long(), exponents.long()) and not scales[:, blocks:].any()
    assert torch.equal(q, packed(codes))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("rows, k", [(1, 32), (3, 64), (1, 16384), (17, 480), (200, 544), (1025, 1056), (4096, 2048)])
def test_quantize(dtype, rows, k):
    x = _randn((rows, k), dtype, 1) * torch.exp2(_randn((rows, 1), torch.float32, 2) * 4).to(dtype)
    _same(x, *_quantize(x))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
def test_quantize_takes_ties_to_the_even_code(dtype):
    """Every value half way between two levels, with a block maximum of 4 to 7.9, in both signs, and zeros of both."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, -0.0, 6.0, 7.0], dtype=torch.float64)
    rows = []
    for largest in (4.0, 4.5, 6.0, 7.0, 7.75):
        for e in (-14, -3, 0, 5):
            row = torch.zeros(32, dtype=torch.float64)
            part = ties[ties <= largest]
            row[:part.numel()] = part
            row[16:16 + part.numel()] = -part
            row[15] = largest
            rows.append(row * 2.0 ** e)
    x = torch.stack(rows).to("cuda", dtype)
    _same(x, *_quantize(x))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
def test_quantize_at_the_ends_of_the_type(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(8, 32, device="cuda", dtype=dtype)
    x[1] = info.max
    x[2] = info.tiny
    x[3, 5] = info.smallest_normal / 4  # below the normal numbers
    x[4, 7] = -info.max
    x[4, 8] = info.tiny
    x[5] = -0.0
    x[6, 0] = info.eps
    x[7] = torch.linspace(-1, 1, 32).to(dtype)
    _same(x, *_quantize(x))


@pytest.mark.parametrize("value", [NAN, float("inf"), -float("inf")])
def test_a_block_with_a_nan_or_an_infinity_is_nan_as_a_whole(value):
    x = torch.ones(2, 96, device="cuda", dtype=torch.bfloat16)
    x[1, 40] = value
    q, scales = _quantize(x)
    _same(x, q, scales)
    out = dequantize_fp4(q, scales, torch.empty_like(x))
    assert out[1, 32:64].isnan().all() and out[0].eq(1).all() and out[1, :32].eq(1).all() and out[1, 64:].eq(1).all()


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("rows, k", [(1, 32), (5, 544), (300, 2048)])
def test_dequantize(dtype, rows, k):
    """Every code under every scale; exact in bf16 and fp32, one rounding in f16."""
    q, scales = operand((rows, k), 1, 0, 255)
    out = dequantize_fp4(q, scales, torch.full((rows, k), NAN, device="cuda", dtype=dtype))
    assert torch.equal(out, values(q, scales).to(dtype))


def test_dequantize_of_all_scales():
    scales = torch.zeros(256, 16, device="cuda", dtype=torch.uint8)
    scales[:, 0] = torch.arange(256)
    q = torch.arange(16, device="cuda", dtype=torch.uint8).mul(0x11).expand(256, 16).contiguous()
    out = dequantize_fp4(q, scales, torch.empty(256, 32, device="cuda"))
    # 4 and 6 times 2^126, and 2 to 6 times 2^127, each in both signs and twice, are above fp32's largest number,
    # just below 2^128: infinite.
    assert torch.equal(out[:255], values(q, scales)[:255].float()) and out[255].isnan().all()
    assert out[:253].isfinite().all() and out[253:255].isinf().sum() == 24


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("tokens, choices, k", [(1, 1, 32), (5, 3, 544), (300, 2, 4096)])
def test_quantize_into_slots(dtype, tokens, choices, k):
    """Each token's row, as quantised alone, in every row its slots name; the other rows as they were."""
    x = _randn((tokens, k), dtype, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = tokens * choices + 3
    slots = torch.randperm(rows, device="cuda", generator=g)[:tokens * choices].view(tokens, choices).to(torch.int32)
    slots[torch.rand(slots.shape, device="cuda", generator=g) < 0.2] = -1
    q = torch.full((rows, k // 2), 0x5a, device="cuda", dtype=torch.uint8)
    scales = torch.full((rows, pitch(k)), 0x5a, device="cuda", dtype=torch.uint8)
    quantize_fp4(x, q, scales, slots=slots)
    want_q, want_scales = _quantize(x)
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for j in range(choices):
        here = slots[:, j] >= 0
        at = slots[here, j].long()
        named[at] = True
        assert torch.equal(q[at], want_q[here]) and torch.equal(scales[at], want_scales[here])
    assert q[~named].eq(0x5a).all() and scales[~named].eq(0x5a).all()


def test_quantize_into_a_slot_behind_the_last_row_is_skipped_and_reported():
    q = torch.zeros(3, 16, device="cuda", dtype=torch.uint8)
    scales = torch.zeros(3, 16, device="cuda", dtype=torch.uint8)
    slots = torch.tensor([[2, 0], [2 ** 31 - 1, 1]], device="cuda", dtype=torch.int32)
    quantize_fp4(torch.ones(2, 32, device="cuda"), q[:2], scales[:2], slots=slots)
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 8
    assert q[:2].eq(0x66).all() and not q[2].any() and not scales[2].any()
    quantize_fp4(torch.ones(2, 32, device="cuda"), q[:0], scales[:0], slots=torch.full_like(slots, -1))


# rows: one, around the steps of 32, below, at and above 128 (a second set of scales) and the largest tile
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 31, 33, 64, 97, 128, 129, 191, 192, 193, 400])
@pytest.mark.parametrize("n, k", [(1, 32), (8, 64), (129, 96), (256, 128), (257, 256), (264, 288), (520, 1056),
                                  (333, 4128)])
def test_product(dtype, rows, n, k):
    a, a_scales = operand((rows, k), 1)
    b, b_scales = operand((n, k), 2, 115, 126)
    out = torch.full((rows, n), NAN, device="cuda", dtype=dtype)
    assert gemm_fp4(a, a_scales, b, b_scales, out) is out
    check(out, *product(values(a, a_scales), values(b, b_scales).unsqueeze(0), [(0, rows)]), k)


# More tiles than the GPU has CTA pairs, so that a pair works through several with its two accumulators; K in one part.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, n, k", [(700, 4100, 288), (1300, 4096, 32), (4100, 4100, 1056), (4095, 4608, 544),
                                        (20000, 264, 1056)])
def test_product_of_many_tiles(dtype, rows, n, k):
    a, a_scales = operand((rows, k), 5)
    b, b_scales = operand((n, k), 6, 115, 126)
    out = torch.full((rows, n), NAN, device="cuda", dtype=dtype)
    gemm_fp4(a, a_scales, b, b_scales, out)
    check(out, *product(values(a, a_scales), values(b, b_scales).unsqueeze(0), [(0, rows)]), k)


# K over clusters of 1, 2, 4 and 8 CTAs (as many as have places at once), tiles of 16 and 64 rows, uneven parts of K.
@pytest.mark.parametrize("rows", [1, 16, 17, 64, 130])
@pytest.mark.parametrize("n, k", [(384, 4640), (2056, 4640), (4096, 1568), (9000, 2080), (18944, 544)])
def test_product_split_over_clusters(rows, n, k):
    a, a_scales = operand((rows, k), 7)
    b, b_scales = operand((n, k), 8, 115, 126)
    out = torch.full((rows, n), NAN, device="cuda", dtype=torch.float16)
    gemm_fp4(a, a_scales, b, b_scales, out)
    check(out, *product(values(a, a_scales), values(b, b_scales).unsqueeze(0), [(0, rows)]), k)


COUNTS = {
    "one_row": [1],
    "one_row_of_many": [0, 0, 1, 0],
    "edges": [31, 32, 33, 0, 191, 192, 193],
    "chunks": [513, 0, 769, 96, 1],
    "many": [(7 * i * i) % 41 for i in range(97)],
    "few_each": [(5 * i) % 12 for i in range(40)],
    "some_each": [(11 * i) % 60 for i in range(9)],
    "uneven": [0, 300, 1, 0, 2, 0, 0, 1],
    "none": [0, 0, 0],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("n, k", [(8, 32), (136, 544), (264, 1024), (777, 352), (1030, 2080)])
def test_product_grouped(dtype, counts, n, k):
    counts = COUNTS[counts]
    rows = sum(counts)
    offsets = offsets_of(counts)
    a, a_scales = operand((rows, k), 3)
    b, b_scales = operand((len(counts), n, k), 4, 115, 126)
    out = torch.full((rows, n), NAN, device="cuda", dtype=dtype)
    gemm_fp4(a, a_scales, b, b_scales, out, offsets=offsets)
    check(out, *product(values(a, a_scales), values(b, b_scales), bounds(offsets)), k)


@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 512, 544, 1024])
def test_each_scale_meets_its_own_values(k):
    """Whole numbers that tell every block of 32, row and column from the others: the products are exact."""
    rows, n = 150, 140
    a = torch.full((rows, k // 2), 0x22, device="cuda", dtype=torch.uint8)  # ones
    b = torch.full((n, k // 2), 0x22, device="cuda", dtype=torch.uint8)
    block = torch.arange(k // 32, device="cuda")
    a_scales = torch.zeros(rows, pitch(k), device="cuda", dtype=torch.uint8)
    b_scales = torch.zeros(n, pitch(k), device="cuda", dtype=torch.uint8)
    a_scales[:, :k // 32] = (127 + (torch.arange(rows, device="cuda").unsqueeze(1) * 3 + block * 5) % 4).byte()
    b_scales[:, :k // 32] = (127 + (torch.arange(n, device="cuda").unsqueeze(1) * 5 + block * 7) % 4).byte()
    out = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    gemm_fp4(a, a_scales, b, b_scales, out)
    want = values(a, a_scales) @ values(b, b_scales).T  # sums of whole numbers below 2^24
    assert torch.equal(out, want.to(torch.float16))


def test_each_value_is_taken_from_its_own_place():
    rows, n, k = 96, 96, 96
    a, a_scales = operand((rows, k), 1, 127, 128)
    eye = torch.zeros(n, k, device="cuda", dtype=torch.long)
    eye[torch.arange(n), torch.arange(k)] = 2  # the code of 1
    out = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    ones = torch.full((n, 16), 127, device="cuda", dtype=torch.uint8)
    gemm_fp4(a, a_scales, packed(eye), ones, out)
    assert torch.equal(out.double(), values(a, a_scales))


def test_what_stands_behind_the_last_scale_does_not_matter():
    rows, n, k = 70, 130, 416
    a, a_scales = operand((rows, k), 1, behind=0)
    b, b_scales = operand((n, k), 2, behind=0)
    out, other = (torch.empty(rows, n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    gemm_fp4(a, a_scales, b, b_scales, out)
    a_scales[:, k // 32:] = 255
    b_scales[:, k // 32:] = 255
    gemm_fp4(a, a_scales, b, b_scales, other)
    assert torch.equal(out, other)


@pytest.mark.parametrize("n", [256, 255])
def test_rows_outside_every_group_are_neither_read_nor_written(n):
    k = 544
    offsets = torch.tensor([5, 40, 40, 260], device="cuda", dtype=torch.int32)
    rows = 300
    a, a_scales = operand((rows, k), 1)
    b, b_scales = operand((3, n, k), 2)
    ref, magnitude = product(values(a, a_scales), values(b, b_scales), bounds(offsets))
    a_scales[:5] = 255  # NaN
    a_scales[260:] = 255
    out = torch.full((rows, n), 7.0, device="cuda", dtype=torch.bfloat16)
    gemm_fp4(a, a_scales, b, b_scales, out, offsets=offsets)
    check(out[5:260], ref[5:260], magnitude[5:260], k)
    assert out[:5].eq(7).all() and out[260:].eq(7).all()


def test_a_nan_scale_makes_its_row_or_column_nan_and_no_other():
    rows, n, k = 140, 300, 704
    a, a_scales = operand((rows, k), 1)
    b, b_scales = operand((n, k), 2)
    ref, magnitude = product(values(a, a_scales), values(b, b_scales).unsqueeze(0), [(0, rows)])
    a_scales[17, 3] = 255
    b_scales[271, 21] = 255
    out = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    gemm_fp4(a, a_scales, b, b_scales, out)
    assert out[17].isnan().all() and out[:, 271].isnan().all()
    out[17], out[:, 271] = ref[17].bfloat16(), ref[:, 271].bfloat16()
    check(out, ref, magnitude, k)


@pytest.mark.parametrize("offsets", [[0, 4, 3], [0, 4, 9], [-1, 4, 8]])
def test_wrong_offsets_compute_nothing_and_are_reported(offsets):
    a, a_scales = operand((8, 64), 1)
    b, b_scales = operand((2, 40, 64), 2)
    out = torch.full((8, 40), 3.0, device="cuda", dtype=torch.bfloat16)
    gemm_fp4(a, a_scales, b, b_scales, out, offsets=torch.tensor(offsets, device="cuda", dtype=torch.int32))
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 7 and out.eq(3).all()


def test_no_rows():
    b, b_scales = operand((40, 64), 2)
    empty = torch.empty(0, 32, device="cuda", dtype=torch.uint8)
    out = torch.empty(0, 40, device="cuda", dtype=torch.bfloat16)
    gemm_fp4(empty, empty[:, :16].contiguous(), b, b_scales, out)
    quantize_fp4(torch.empty(0, 64, device="cuda"), empty, empty[:, :16].contiguous())
    dequantize_fp4(empty, empty[:, :16].contiguous(), torch.empty(0, 64, device="cuda"))


def test_repeats_bit_for_bit_on_two_streams_at_once():
    rows, n, k = 700, 1000, 2048
    a, a_scales = operand((rows, k), 1)
    b, b_scales = operand((n, k), 2)
    outs = [torch.empty(rows, n, device="cuda", dtype=torch.bfloat16) for _ in range(5)]
    gemm_fp4(a, a_scales, b, b_scales, outs[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i, out in enumerate(outs[1:]):
        streams[i % 2].wait_stream(torch.cuda.current_stream())
        gemm_fp4(a, a_scales, b, b_scales, out, stream=streams[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], out) for out in outs[1:])


def test_an_expert_layer_in_4_bits_in_a_graph():
    """sort, quantise into slots, product and combine as one captured step, replayed on other choices and rows."""
    tokens, choices, experts, k, n = 77, 3, 8, 544, 264
    rows = tokens * choices
    x = _randn((tokens, k), torch.bfloat16, 1)
    b, b_scales = operand((experts, n, k), 2, 118, 121)
    w = torch.softmax(_randn((tokens, choices), torch.float32, 3), 1)
    ids = torch.zeros(tokens, choices, device="cuda", dtype=torch.int64)
    offsets = torch.empty(experts + 1, device="cuda", dtype=torch.int32)
    slots = torch.empty(tokens, choices, device="cuda", dtype=torch.int32)
    a = torch.empty(rows, k // 2, device="cuda", dtype=torch.uint8)
    a_scales = torch.empty(rows, pitch(k), device="cuda", dtype=torch.uint8)
    y = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    out = torch.empty(tokens, n, device="cuda", dtype=torch.bfloat16)

    def step():
        expert_sort(ids, offsets, slots)
        quantize_fp4(x, a, a_scales, slots=slots)
        gemm_fp4(a, a_scales, b, b_scales, y, offsets=offsets)
        expert_combine(y, slots, out, weights=w)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    weights = values(b, b_scales)
    for seed in (4, 5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        ids.copy_(torch.randint(-1, experts, ids.shape, device="cuda", generator=g))
        x.copy_(_randn(x.shape, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        codes, exponents = quantised(x)
        padded = torch.zeros(tokens, pitch(k), device="cuda", dtype=torch.uint8)
        padded[:, :k // 32] = exponents
        xq = values(packed(codes), padded)
        here = (ids >= 0).unsqueeze(-1)
        chosen = weights[ids.clamp_min(0)]
        exact = [torch.where(here, torch.einsum("tk,tjnk->tjn", f(xq), f(chosen)), 0.0) * w.double().unsqueeze(-1)
                 for f in (lambda t: t, torch.abs)]
        # Two roundings to bf16 and sums of k + choices terms in fp32, of at most the sum of absolute values.
        share = (1 + 2.0 ** -8) ** 2 - 1 + 2 * (k + choices + 16) * 2.0 ** -23
        assert ((out.double() - exact[0].sum(1)).abs() <= share * exact[1].sum(1)).all()
