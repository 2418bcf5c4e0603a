"""GPU tests of rows to the experts and back (expert_sort, expert_dispatch, expert_combine, expert_combine_grad) against
plain 64-bit forms, with elementwise bounds derived from the number formats."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import (  # noqa: E402
    expert_combine, expert_combine_grad, expert_dispatch, expert_sort, grouped_gemm, grouped_gemm_wgrad)

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
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


def _ids(tokens, choices, experts, seed, outside=0.0, dtype=torch.int64):
    """Any experts, one twice a token too; a share of them outside [0, experts) on both sides."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, choices), device="cuda", generator=g)
    gone = torch.rand(ids.shape, device="cuda", generator=g) < outside
    wrong = torch.where(torch.rand(ids.shape, device="cuda", generator=g) < 0.5, -1, experts)
    return torch.where(gone, wrong, ids).to(dtype)


def _sorted(ids, experts):
    flat = ids.reshape(-1).long().cpu()
    slots = torch.full_like(flat, -1)
    offsets, at = [0], 0
    for e in range(experts):
        mine = (flat == e).nonzero().squeeze(1)
        slots[mine] = torch.arange(at, at + mine.numel())
        at += mine.numel()
        offsets.append(at)
    return torch.tensor(offsets, dtype=torch.int32), slots.reshape(ids.shape).to(torch.int32)


def _sort(ids, experts):
    return expert_sort(ids, torch.full((experts + 1,), -7, device="cuda", dtype=torch.int32),
                       torch.full(ids.shape, -7, device="cuda", dtype=torch.int32))


# tokens and choices: none, one, around a warp's 32 and a CTA's 1024, over one, four and eight CTAs
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens, choices", [(0, 2), (1, 1), (1, 8), (31, 1), (33, 1), (1023, 2), (1025, 1), (2049, 1),
                                             (1500, 5), (8191, 4), (40000, 3)])
@pytest.mark.parametrize("experts, outside", [(1, 0.0), (8, 0.3), (257, 0.0), (1024, 0.9)])
def test_sort(dtype, tokens, choices, experts, outside):
    ids = _ids(tokens, choices, experts, 1, outside, dtype)
    offsets, slots = _sort(ids, experts)
    want_offsets, want_slots = _sorted(ids, experts)
    assert torch.equal(offsets.cpu(), want_offsets) and torch.equal(slots.cpu(), want_slots)


@pytest.mark.parametrize("value", [3, -1, 2 ** 31 - 1])
def test_sort_with_one_expert_for_all(value):
    ids = torch.full((5000, 2), value, device="cuda", dtype=torch.int32)
    offsets, slots = _sort(ids, 8)
    want_offsets, want_slots = _sorted(ids, 8)
    assert torch.equal(offsets.cpu(), want_offsets) and torch.equal(slots.cpu(), want_slots)


def test_sort_takes_int64_whole():
    """An id whose low 32 bits name an expert is none."""
    ids = torch.tensor([[2 ** 32 + 1, 1], [-(2 ** 32), 0]], device="cuda")
    offsets, slots = _sort(ids, 2)
    assert offsets.tolist() == [0, 1, 2] and slots.tolist() == [[-1, 1], [-1, 0]]


# Half a step of a type, relative to the value, and half of its smallest number.
HALF = {d: torch.finfo(d).eps / 2 for d in DTYPES.values()}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _close(got, ref, magnitude, terms):
    """One rounding to got's type of a sum of `terms` fp32 products: each product and each add drops at most 2^-24 of
    itself, and no partial sum is above `magnitude` (the sum of the absolute products) by more than those errors."""
    err = 2 * (terms + 1) * 2.0 ** -24 * magnitude
    bound = err + HALF[got.dtype] * (ref.abs() + err) + TINY[got.dtype]
    excess = (got.double() - ref).abs() - bound
    assert not (excess > 0).any() and not got.isnan().any(), excess.max().item()


def _plan(tokens, choices, experts=6, outside=0.25, seed=3):
    ids = _ids(tokens, choices, experts, seed, outside)
    offsets, slots = _sort(ids, experts)
    return offsets, slots, (slots >= 0)


# widths: one value, no vector, one vector of 16 bytes and one value more, rows of 2-, 4-, 8- and 16-byte accesses, more
# than a CTA takes at once
WIDTHS = [1, 7, 8, 9, 1001, 1002, 1004, 2048, 4104]
TOKENS = [(1, 1), (1, 9), (3, 2), (130, 4), (1201, 5)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("weights", [None, "own", "float32"])
@pytest.mark.parametrize("tokens, choices", TOKENS)
@pytest.mark.parametrize("width", WIDTHS)
def test_dispatch(dtype, weights, tokens, choices, width):
    _, slots, here = _plan(tokens, choices)
    x = _randn((tokens, width), dtype, 1)
    w = None if weights is None else _randn((tokens, choices), dtype if weights == "own" else torch.float32, 2)
    rows = tokens * choices + 3
    out = torch.full((rows, width), NAN, device="cuda", dtype=dtype)
    assert expert_dispatch(x, slots, out, weights=w) is out
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    named[slots[here].long()] = True
    assert out[~named].isnan().all()
    values = x.unsqueeze(1).expand(-1, choices, -1)[here]
    if w is None:
        assert torch.equal(out[slots[here].long()], values)
    else:
        ref = values.double() * w[here].double().unsqueeze(1)
        _close(out[slots[here].long()], ref, ref.abs(), 1)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("weights", [None, "own", "float32"])
@pytest.mark.parametrize("tokens, choices", TOKENS)
@pytest.mark.parametrize("width", WIDTHS)
def test_combine(dtype, weights, tokens, choices, width):
    _, slots, here = _plan(tokens, choices)
    y = _randn((tokens * choices + 1, width), dtype, 1)
    y[int(here.sum()):] = NAN  # rows that no slot names
    w = None if weights is None else _randn((tokens, choices), dtype if weights == "own" else torch.float32, 2)
    out = torch.full((tokens, width), NAN, device="cuda", dtype=dtype)
    assert expert_combine(y, slots, out, weights=w) is out
    terms = torch.where(here.unsqueeze(-1), y[slots.clamp_min(0).long()].double(), 0.0)
    if w is not None:
        terms = terms * w.double().unsqueeze(-1)
    _close(out, terms.sum(1), terms.abs().sum(1), choices)
    assert not out[~here.any(1)].any()


def _grad_reference(grad, y, slots, here, w):
    rows = y[slots.clamp_min(0).long()].double()
    products = torch.where(here.unsqueeze(-1), grad.double().unsqueeze(1) * rows, 0.0)
    return grad.double().unsqueeze(1) * w.double().unsqueeze(-1), products.sum(-1), products.abs().sum(-1)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("weights", ["own", "float32"])
@pytest.mark.parametrize("tokens, choices", TOKENS)
@pytest.mark.parametrize("width", WIDTHS)
def test_combine_grad(dtype, weights, tokens, choices, width):
    _, slots, here = _plan(tokens, choices)
    rows = tokens * choices + 2
    y, grad = _randn((rows, width), dtype, 1), _randn((tokens, width), dtype, 2)
    y[int(here.sum()):] = NAN
    w = _randn((tokens, choices), dtype if weights == "own" else torch.float32, 3)
    grad_y, grad_w = torch.full_like(y, NAN), torch.full_like(w, NAN)
    assert expert_combine_grad(grad, y, slots, w, grad_y, grad_w) == (grad_y, grad_w)
    ref_y, ref_w, magnitude = _grad_reference(grad, y, slots, here, w)
    _close(grad_y[slots[here].long()], ref_y[here], ref_y[here].abs(), 1)
    _close(grad_w, ref_w, magnitude, width)
    assert grad_y[int(here.sum()):].isnan().all() and not grad_w[~here].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
@pytest.mark.parametrize("tokens, choices, packs", [(4737, 1, 1), (4800, 3, 31), (9600, 5, 33), (5003, 9, 255), (4736, 2, 64),
                                                   (148, 4, 256), (700, 9, 257), (593, 1, 511), (1300, 2, 512),
                                                   (1185, 7, 300)])
def test_combine_grad_of_many_tokens(dtype, tokens, choices, packs):
    """A warp's and a CTA's tokens: rows of 16-byte packs around a warp's, a CTA's and a ring's, tokens in one go and more."""
    width = packs * (16 // dtype.itemsize)
    _, slots, here = _plan(tokens, choices)
    rows = int(here.sum()) + 2
    y, grad = _randn((rows, width), dtype, 1), _randn((tokens, width), dtype, 2)
    y[-2:] = NAN
    w = _randn((tokens, choices), torch.float32, 3)
    w[~here] = NAN
    grad_y, grad_w, in_place, again = torch.full_like(y, NAN), torch.full_like(w, NAN), y.clone(), torch.empty_like(w)
    expert_combine_grad(grad, y, slots, w, grad_y, grad_w)
    for lo in range(0, tokens, 1000):
        part = slice(lo, lo + 1000)
        ref_y, ref_w, magnitude = _grad_reference(grad[part], y, slots[part], here[part], w[part])
        at = here[part]
        _close(grad_y[slots[part][at].long()], ref_y[at], ref_y[at].abs(), 1)
        _close(grad_w[part], ref_w, magnitude, width)
    assert grad_y[-2:].isnan().all() and not grad_w[~here].any()
    expert_combine_grad(grad, in_place, slots, w, in_place, again)
    assert torch.equal(in_place[:-2], grad_y[:-2]) and torch.equal(again, grad_w)


def test_gradients_agree_with_differences():
    """<combine_grad, direction> against the difference of two 64-bit combines along it; combine is linear in each."""
    tokens, choices, width = 7, 3, 40
    _, slots, here = _plan(tokens, choices, outside=0.2)
    y, w = _randn((tokens * choices, width), torch.float32, 1), _randn((tokens, choices), torch.float32, 2)
    grad = _randn((tokens, width), torch.float32, 3)
    grad_y, grad_w, grad_x = torch.zeros_like(y), torch.zeros_like(w), torch.zeros_like(grad)
    expert_combine_grad(grad, y, slots, w, grad_y, grad_w)
    rows = _randn(y.shape, torch.float32, 6)
    expert_combine(rows, slots, grad_x, weights=w)

    def loss(y, w):
        terms = torch.where(here.unsqueeze(-1), y[slots.clamp_min(0).long()], 0.0) * w.unsqueeze(-1)
        return (terms.sum(1) * grad.double()).sum()

    def dispatched(x):
        out = torch.zeros(y.shape, device="cuda", dtype=torch.float64)
        out[slots[here].long()] = (x.unsqueeze(1) * w.double().unsqueeze(-1))[here]
        return (out * rows.double()).sum()

    dy, dw, dx = _randn(y.shape, torch.float64, 4), _randn(w.shape, torch.float64, 5), _randn(grad.shape, torch.float64, 7)
    x0 = _randn(grad.shape, torch.float64, 8)
    for got, step, difference in (
            (grad_y, dy, loss(y.double() + dy, w.double()) - loss(y.double(), w.double())),
            (grad_w, dw, loss(y.double(), w.double() + dw) - loss(y.double(), w.double())),
            (grad_x, dx, dispatched(x0 + dx) - dispatched(x0))):
        # each of the entries of `got` is off by at most (width + 2) fp32 roundings of a sum of products below 20 * width
        assert (got.double() * step).sum().sub(difference).abs() <= 20 * width * (width + 2) * 2.0 ** -24 * step.abs().sum()


def test_values_of_rows_that_are_not_there_do_not_matter():
    """A weight of a choice without a row, infinite or NaN, counts for nothing; a row's own infinities stay."""
    slots = torch.tensor([[0, -1], [-1, -1], [-3, 1]], device="cuda", dtype=torch.int32)
    w = torch.tensor([[1.0, NAN], [NAN, float("inf")], [NAN, 2.0]], device="cuda")
    y = torch.ones(2, 16, device="cuda")
    y[1, 3] = float("inf")
    out = torch.full((3, 16), NAN, device="cuda")
    expert_combine(y, slots, out, weights=w)
    assert out[0].eq(1).all() and out[1].eq(0).all() and out[2, 3].isinf() and out[2, 4:].eq(2).all()
    grad_y, grad_w = torch.full_like(y, NAN), torch.full_like(w, NAN)
    expert_combine_grad(torch.ones(3, 16, device="cuda"), y, slots, w, grad_y, grad_w)
    assert grad_y[0].eq(1).all() and grad_y[1].eq(2).all()
    assert grad_w[:, 0].tolist() == [16.0, 0.0, 0.0] and grad_w[:2, 1].tolist() == [0.0, 0.0] and grad_w[2, 1].isinf()


@pytest.mark.parametrize("width", [8, 9])
def test_a_slot_behind_the_last_row_is_skipped_and_reported(width):
    slots = torch.tensor([[0, 4], [2 ** 31 - 1, 1]], device="cuda", dtype=torch.int32)
    x, w = torch.ones(2, width, device="cuda"), torch.ones(2, 2, device="cuda")
    rows = torch.zeros(5, width, device="cuda")[:4]
    guard = rows.untyped_storage()
    for call in (lambda: expert_dispatch(x, slots, rows), lambda: expert_combine(rows, slots, x),
                 lambda: expert_combine_grad(x, rows, slots, w, rows, torch.empty_like(w))):
        call()
        torch.cuda.synchronize()
        assert _native.device_error(0, clear=True) == 8
    whole = torch.empty(0, device="cuda").set_(guard, 0, (5, width))
    assert rows[0].eq(1).all() and rows[1].eq(1).all() and not whole[2:].any()


def _at(t, offset):
    """A copy of t that begins `offset` values behind an aligned address, with NaN around it."""
    whole = torch.full((t.numel() + 32,), float("nan"), device="cuda", dtype=t.dtype)
    there = whole[offset:offset + t.numel()].view(t.shape)
    there.copy_(t)
    return whole, there


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 255, 256, 257, 510, 2046, 2048])
@pytest.mark.parametrize("offsets", [(0, 1), (1, 0), (1, 1), (2, 1), (3, 2), (4, 7), (5, 3), (6, 6), (7, 4)])
def test_rows_that_begin_anywhere(dtype, width, offsets):
    """Every place of a row in 16 bytes; rows that no slot names, and all around the matrices, are NaN and stay so."""
    tokens, choices = 37, 5
    _, slots, here = _plan(tokens, choices)
    count = int(here.sum())
    slots = torch.where(here, 2 * slots, -1)  # every other row of 2 * count - 1
    g = torch.Generator(device="cuda").manual_seed(width)
    rows = torch.full((2 * count - 1, width), float("nan"), device="cuda", dtype=dtype)
    rows[::2] = torch.randn(count, width, generator=g, device="cuda").to(dtype)
    x = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
    w = torch.randn(tokens, choices, generator=g, device="cuda")
    around_y, y = _at(rows, offsets[0])
    around_out, out = _at(torch.zeros_like(x), offsets[1])
    expert_combine(y, slots, out, weights=w)
    want = torch.zeros_like(x, dtype=torch.float32)
    for j in range(choices):  # fp32, in the order of the choices: fma's one rounding less is what differs
        want += torch.where(here[:, j:j + 1], w[:, j:j + 1] * rows[slots[:, j].clamp_min(0).long()].float(), 0.0)
    size = torch.stack([torch.where(here[:, j:j + 1], (w[:, j:j + 1] * rows[slots[:, j].clamp_min(0).long()].float()).abs(),
                                    0.0) for j in range(choices)]).sum(0)
    eps = torch.finfo(dtype).eps / 2
    assert ((out.double() - want.double()).abs() <= eps * want.double().abs() + 4 * choices * 2.0 ** -24 * size.double()).all()
    assert around_out.isnan().sum() == 32
    around_x, xs = _at(x, offsets[0])
    around_rows, ys = _at(torch.full_like(rows, float("nan")), offsets[1])
    expert_dispatch(xs, slots, ys)
    assert torch.equal(ys[slots[here].long()], x.unsqueeze(1).expand(-1, choices, -1)[here])
    assert ys[1::2].isnan().all() and around_rows.isnan().sum() == 32 + (count - 1) * width
    grad_w = torch.empty_like(w)
    around_rows, gy = _at(torch.full_like(rows, float("nan")), offsets[1])
    expert_combine_grad(xs, y, slots, w, gy, grad_w)
    assert torch.equal(gy[slots[here].long()], (w.unsqueeze(-1) * x.float().unsqueeze(1))[here].to(dtype))
    assert gy[1::2].isnan().all() and around_rows.isnan().sum() == 32 + (count - 1) * width
    products = x.double().unsqueeze(1) * rows[slots.clamp_min(0).long()].double()
    want_w = torch.where(here, products.sum(-1), 0.0)
    slack = torch.where(here, products.abs().sum(-1), 0.0) * width * 2.0 ** -24
    assert ((grad_w.double() - want_w).abs() <= slack + 2.0 ** -24 * want_w.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width, choices", [(264, 6), (263, 6), (2048, 4), (8, 1), (1, 2), (6, 9)])
def test_gradient_into_y_itself(dtype, width, choices):
    _, slots, here = _plan(300, choices)
    g = torch.Generator(device="cuda").manual_seed(width)
    grad, y = (torch.randn(n, width, generator=g, device="cuda").to(dtype) for n in (300, int(here.sum()) + 3))
    w = torch.randn(300, choices, generator=g, device="cuda")
    apart, weights_apart, weights_same = y.clone(), torch.empty_like(w), torch.empty_like(w)
    expert_combine_grad(grad, y, slots, w, apart, weights_apart)
    expert_combine_grad(grad, y, slots, w, y, weights_same)
    assert torch.equal(y, apart) and torch.equal(weights_same, weights_apart)


def test_sort_into_the_choices_themselves_is_refused():
    ids = torch.zeros(50, 2, device="cuda", dtype=torch.int32)
    with pytest.raises(_native.NativeError, match="must not overlap"):
        expert_sort(ids, torch.empty(9, device="cuda", dtype=torch.int32), ids)
    x = torch.ones(4, 32, device="cuda")
    with pytest.raises(_native.NativeError, match="must not overlap"):
        expert_dispatch(x, torch.zeros(4, 1, device="cuda", dtype=torch.int32), x)
    assert not ids.any() and x.eq(1).all()


def test_nothing_to_do():
    empty = torch.empty(0, 2, device="cuda", dtype=torch.int32)
    x = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16)
    rows = torch.ones(3, 16, device="cuda", dtype=torch.bfloat16)
    expert_dispatch(x, empty, rows)
    expert_combine(rows, empty, x)
    w = torch.empty(0, 2, device="cuda")
    expert_combine_grad(x, rows, empty, w, rows, w)
    assert rows.eq(1).all()
    slots = torch.full((4, 2), -1, device="cuda", dtype=torch.int32)
    out = torch.ones(4, 16, device="cuda", dtype=torch.bfloat16)
    expert_combine(x, slots, out)  # no rows at all: zeros
    assert not out.any()
    expert_dispatch(out, slots, x)


def test_calls_repeat_bit_for_bit_and_unaligned_rows_give_the_same():
    _, slots, _ = _plan(300, 6)
    width = 264
    y, grad = _randn((1800, width), torch.bfloat16, 1), _randn((300, width), torch.bfloat16, 2)
    w = _randn((300, 6), torch.float32, 3)

    def all_of(y, grad):
        out, grad_y, grad_w = torch.zeros_like(grad), torch.zeros_like(y), torch.zeros_like(w)
        expert_combine(y, slots, out, weights=w)
        expert_combine_grad(grad, y, slots, w, grad_y, grad_w)
        return out, grad_y, grad_w

    first = all_of(y, grad)
    assert all(torch.equal(a, b) for a, b in zip(first, all_of(y, grad)))

    def shifted(t):
        buffer = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        return buffer[1:].view(t.shape).copy_(t)

    out, grad_y = shifted(grad), shifted(torch.zeros_like(y))
    grad_w = torch.empty_like(w)
    expert_combine(shifted(y), slots, out, weights=w)
    expert_combine_grad(shifted(grad), shifted(y), slots, w, grad_y, grad_w)
    assert torch.equal(out, first[0]) and torch.equal(grad_y, first[1])
    torch.testing.assert_close(grad_w, first[2], rtol=0, atol=2 * 264 * 2.0 ** -24 * 300)  # another order of 264 products


def test_a_layer_and_its_gradients_on_a_stream_and_in_a_graph():
    """sort, dispatch, product, combine and all gradients as one captured step, replayed on other choices."""
    tokens, choices, experts, k, n = 90, 2, 8, 64, 48
    x = _randn((tokens, k), torch.bfloat16, 1)
    b = (_randn((experts, k, n), torch.float32, 2) * k ** -0.5).to(torch.bfloat16)
    w = torch.softmax(_randn((tokens, choices), torch.float32, 3), 1)
    grad = _randn((tokens, n), torch.bfloat16, 4)
    ids = _ids(tokens, choices, experts, 5)
    rows = tokens * choices
    new = dict(device="cuda", dtype=torch.bfloat16)
    offsets = torch.empty(experts + 1, device="cuda", dtype=torch.int32)
    slots = torch.empty(tokens, choices, device="cuda", dtype=torch.int32)
    xs, ys, out = torch.zeros(rows, k, **new), torch.zeros(rows, n, **new), torch.empty(tokens, n, **new)
    gy, gw, gxs, gx, gb = torch.zeros_like(ys), torch.empty_like(w), torch.zeros_like(xs), torch.empty_like(x), torch.empty_like(b)

    def step():
        expert_sort(ids, offsets, slots)
        expert_dispatch(x, slots, xs)
        grouped_gemm(xs, b, offsets, ys)
        expert_combine(ys, slots, out, weights=w)
        expert_combine_grad(grad, ys, slots, w, gy, gw)
        grouped_gemm(gy, b, offsets, gxs, b_transposed=True)
        grouped_gemm_wgrad(xs, gy, offsets, gb)
        expert_combine(gxs, slots, gx)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed, outside in ((6, 0.0), (7, 0.5), (8, 1.0)):
        ids.copy_(_ids(tokens, choices, experts, seed, outside))
        graph.replay()
        torch.cuda.synchronize()
        here = (ids >= 0) & (ids < experts)

        def exact(x, b, w, grad):
            x, b, w = (t.double().requires_grad_() for t in (x, b, w))
            y = torch.einsum("tk,tjkn->tjn", x, b[ids.clamp(0, experts - 1)])
            y = torch.where(here.unsqueeze(-1), y, 0.0)
            out = (y * w.unsqueeze(-1)).sum(1)
            return out.detach(), *torch.autograd.grad((out * grad.double()).sum(), (x, b, w))

        # Everything here is sums of products of inputs.  A result that went through r roundings to bf16, and sums of at
        # most rows + k + n + 16 terms in fp32, is off by at most that share of the same sums of absolute values.
        sums = (rows + k + n + 16) * 2.0 ** -23
        for got, want, magnitude, r in zip((out, gx, gb, gw), exact(x, b, w, grad),
                                           exact(x.abs(), b.abs(), w, grad.abs()), (2, 3, 2, 1)):
            share = (1 + 2.0 ** -8) ** r - 1 + 2 * sums
            assert ((got.double() - want).abs() <= share * magnitude).all()
