"""Host side of rows to the experts and back and of 4-bit floating point: the C entry points' refusals, the front ends'
checks and the device that they launch on, none of which needs a GPU."""
from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200 import _native, kernels  # noqa: E402
from tests.test_kernels_device import Stub  # noqa: E402

BF16, F16, F32, F64 = 1, 2, 0, 3
P = 4096  # an aligned address that is never read: every call below is refused first, or has nothing to do
LARGEST = 2130706432


@pytest.mark.parametrize("args, status, message", [
    ((4, -1, 2, 8, P, P, P, None), -1, "sizes must be positive"),
    ((4, 1, 0, 8, P, P, P, None), -1, "sizes must be positive"),
    ((4, 1, 2, 0, P, P, P, None), -1, "sizes must be positive"),
    ((4, 1, 2, 8, None, P, P, None), -1, "non-null"),
    ((4, 1, 2, 8, P, P, None, None), -1, "non-null"),
    ((4, 0, 2, 8, None, None, None, None), -1, "non-null"),
    ((2, 1, 2, 8, P, P, P, None), 1, "int32 or int64"),
    ((8, 1, 2, 1025, P, P, P, None), 1, "at most 1024 experts"),
    ((8, LARGEST // 2 + 1, 2, 8, P, P, P, None), 1, f"at most {LARGEST}"),
    ((8, 1, 2, 8, P + 4, P, P, None), -3, "aligned"),
    ((4, 1, 2, 8, P, P + 2, P, None), -3, "aligned"),
])
def test_sort_entry(args, status, message):
    assert _native.load().trb_expert_sort_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("entry", ["trb_expert_dispatch_launch", "trb_expert_combine_launch"])
@pytest.mark.parametrize("args, status, message", [
    ((BF16, F32, -1, 2, 4, 8, P, P, P, P, None), -1, "sizes must be positive"),
    ((BF16, F32, 1, 0, 4, 8, P, P, P, P, None), -1, "sizes must be positive"),
    ((BF16, F32, 1, 2, 4, 0, P, P, P, P, None), -1, "sizes must be positive"),
    ((BF16, F32, 1, 2, 4, 8, P, None, P, P, None), -1, "non-null"),
    ((BF16, F32, 1, 2, 4, 8, None, P, P, P, None), -1, "non-null"),
    ((BF16, F32, 1, 2, 4, 8, P, P, P, None, None), -1, "non-null"),
    ((F64, F32, 1, 2, 4, 8, P, P, P, P, None), 1, "unsupported dtype"),
    ((BF16, F16, 1, 2, 4, 8, P, P, P, P, None), 1, "weights must be"),
    ((BF16, F32, 1, 2, LARGEST + 1, 8, P, P, P, P, None), 1, f"at most {LARGEST}"),
    ((BF16, F32, LARGEST, 2, 4, 8, P, P, P, P, None), 1, f"at most {LARGEST}"),
    ((BF16, F32, 1, 2, 4, 8, P + 1, P, P, P, None), -3, "aligned"),
    ((BF16, F32, 1, 2, 4, 8, P, P + 2, P, P, None), -3, "aligned"),
    ((BF16, F32, 1, 2, 4, 8, P, P, P + 2, P, None), -3, "aligned"),
    ((BF16, F32, 0, 2, 4, 8, None, None, None, P, None), 0, ""),
])
def test_dispatch_and_combine_entries(entry, args, status, message):
    assert getattr(_native.load(), entry)(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("args, status, message", [
    ((BF16, F32, 1, 2, 4, 8, None, P, P, P, P, P, None), -1, "non-null"),
    ((BF16, F32, 1, 2, 4, 8, P, P, P, None, P, P, None), -1, "non-null"),
    ((BF16, F32, 1, 2, 4, 8, P, P, P, P, None, P, None), -1, "non-null"),
    ((BF16, F32, 1, 2, 4, 8, P, P, P, P, P, None, None), -1, "non-null"),
    ((BF16, F64, 1, 2, 4, 8, P, P, P, P, P, P, None), 1, "weights must be"),
    ((F32, F32, 1, 2, 4, 8, P + 2, P, P, P, P, P, None), -3, "aligned"),
    ((BF16, F32, 1, 2, 4, 8, P, P, P, P, P, P + 2, None), -3, "aligned"),
    ((BF16, F32, 0, 2, 4, 8, None, P, None, None, P, None, None), 0, ""),
])
def test_combine_grad_entry(args, status, message):
    assert _native.load().trb_expert_combine_grad_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("args, status, message", [
    ((BF16, -1, 64, P, 1, None, 0, P, P, None), -1, "sizes must be positive"),
    ((BF16, 4, 0, P, 1, None, 0, P, P, None), -1, "sizes must be positive"),
    ((F64, 4, 64, P, 1, None, 0, P, P, None), 1, "unsupported dtype"),
    ((BF16, LARGEST + 1, 64, P, 1, None, 0, P, P, None), 1, f"at most {LARGEST}"),
    ((BF16, 4, 48, P, 1, None, 0, P, P, None), -3, "multiple of 32"),
    ((BF16, 4, 64, None, 1, None, 0, P, P, None), -1, "non-null"),
    ((BF16, 4, 64, P, 1, None, 0, P, None, None), -1, "non-null"),
    ((BF16, 4, 64, P + 8, 1, None, 0, P, P, None), -3, "16-byte aligned"),
    ((BF16, 4, 64, P, 1, None, 0, P, P + 1, None), -3, "16-byte aligned"),
    ((BF16, 4, 64, P, 0, P, 8, P, P, None), -1, "slots need choices"),
    ((BF16, 4, 64, P, 1, P + 2, 8, P, P, None), -1, "slots need choices"),
    ((BF16, 4, 64, P, 1, P, LARGEST + 1, P, P, None), 1, f"at most {LARGEST}"),
    ((BF16, LARGEST, 64, P, 2, P, 8, P, P, None), 1, f"at most {LARGEST}"),
    ((BF16, 0, 64, None, 1, None, 0, None, None, None), 0, ""),
])
def test_quantize_entry(args, status, message):
    assert _native.load().trb_quantize_fp4_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("args, status, message", [
    ((F64, 4, 64, P, P, P, None), 1, "unsupported dtype"),
    ((BF16, 4, 33, P, P, P, None), -3, "multiple of 32"),
    ((BF16, 4, 64, P, P, None, None), -1, "non-null"),
    ((BF16, 4, 64, P, P, P + 4, None), -3, "16-byte aligned"),
    ((BF16, 0, 64, None, None, None, None), 0, ""),
])
def test_dequantize_entry(args, status, message):
    assert _native.load().trb_dequantize_fp4_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("args, status, message", [
    ((BF16, 0, 4, 8, 64, P, P, P, P, P, P, None), -1, "sizes must be positive"),
    ((BF16, 1, 4, 0, 64, P, P, P, P, P, P, None), -1, "sizes must be positive"),
    ((BF16, 2, 4, 8, 64, P, P, P, P, None, P, None), -1, "several groups need offsets"),
    ((F32, 1, 4, 8, 64, P, P, P, P, None, P, None), 1, "unsupported dtype"),
    ((BF16, 1025, 4, 8, 64, P, P, P, P, P, P, None), 1, "at most 1024 groups"),
    ((BF16, 1, LARGEST + 1, 8, 64, P, P, P, P, None, P, None), 1, f"at most {LARGEST}"),
    ((BF16, 1, 4, 8, 2 ** 26 + 32, P, P, P, P, None, P, None), 1, f"k at most {2 ** 26}"),
    ((BF16, 1, 4, 8, 40, P, P, P, P, None, P, None), -3, "multiple of 32"),
    ((BF16, 1, 4, 8, 64, P, None, P, P, None, P, None), -1, "non-null"),
    ((BF16, 1, 4, 8, 64, P, P, P, P + 8, None, P, None), -3, "16-byte aligned"),
    ((BF16, 1, 4, 8, 64, P, P, P, P, P + 2, P, None), -3, "4-byte aligned"),
    ((BF16, 1, 0, 8, 64, None, None, None, None, None, None, None), 0, ""),
])
def test_gemm_fp4_entry(args, status, message):
    assert _native.load().trb_gemm_fp4_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("launch, sizes", [
    (lambda *s: _native.expert_sort_launch(8, *s, P, P, P), 3),
    (lambda *s: _native.expert_dispatch_launch("bfloat16", "float32", *s, P, P, P, P), 4),
    (lambda *s: _native.expert_combine_launch("bfloat16", "float32", *s, P, P, P, P), 4),
    (lambda *s: _native.expert_combine_grad_launch("bfloat16", "float32", *s, P, P, P, P, P, P), 4),
    (lambda rows, k, c, o: _native.quantize_fp4_launch("bfloat16", rows, k, P, c, P, o, P, P), 4),
    (lambda *s: _native.dequantize_fp4_launch("bfloat16", *s, P, P, P), 2),
    (lambda *s: _native.gemm_fp4_launch("bfloat16", *s, P, P, P, P, P, P), 4),
], ids=["sort", "dispatch", "combine", "combine_grad", "quantize", "dequantize", "gemm"])
def test_sizes_past_32_bits_are_not_cut(launch, sizes):
    for i in range(sizes):
        args = [64] * sizes
        args[i] += 2 ** 32
        with pytest.raises(ValueError, match="32 bits"):
            launch(*args)


I32, U8 = torch.int32, torch.uint8
SLOTS, X, ROWS, W = Stub(4, 2, dtype=I32), Stub(4, 64), Stub(8, 64), Stub(4, 2, dtype=torch.float32)
Q, SCALES = Stub(8, 32, dtype=U8), Stub(8, 16, dtype=U8)
CALLS = {
    "expert_sort_launch": lambda **kw: kernels.expert_sort(Stub(4, 2, dtype=torch.int64), Stub(9, dtype=I32), SLOTS, **kw),
    "expert_dispatch_launch": lambda **kw: kernels.expert_dispatch(X, SLOTS, ROWS, **kw),
    "expert_combine_launch": lambda **kw: kernels.expert_combine(ROWS, SLOTS, X, weights=W, **kw),
    "expert_combine_grad_launch": lambda **kw: kernels.expert_combine_grad(X, ROWS, SLOTS, W, ROWS, W, **kw),
    "quantize_fp4_launch": lambda **kw: kernels.quantize_fp4(X, Q, SCALES, slots=SLOTS, **kw),
    "dequantize_fp4_launch": lambda **kw: kernels.dequantize_fp4(Q, SCALES, ROWS, **kw),
    "gemm_fp4_launch": lambda **kw: kernels.gemm_fp4(Q, SCALES, Stub(3, 5, 32, dtype=U8), Stub(3, 5, 16, dtype=U8),
                                                     Stub(8, 5), offsets=Stub(4, dtype=I32), **kw),
}


@pytest.fixture
def machine(monkeypatch):
    """Two devices, of which the thread's current one is 0; `launched` holds the current device at each launch."""
    m = types.SimpleNamespace(current=0, launched=[])

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, m.current = m.current, self.index

        def __exit__(self, *_):
            m.current = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(kernels, "_CURRENT_DEVICE", lambda: m.current)
    monkeypatch.setattr(kernels, "_RAW_STREAM", lambda index: 0)
    for name in CALLS:
        monkeypatch.setattr(_native, name, lambda *args: m.launched.append(m.current))
    return m


@pytest.mark.parametrize("call", CALLS)
def test_launches_on_the_tensors_device_and_refuses_another_stream(machine, call):
    CALLS[call]()
    assert machine.launched == [1] and machine.current == 0
    with pytest.raises(ValueError, match="stream is on cuda:0"):
        CALLS[call](stream=types.SimpleNamespace(cuda_stream=0, device_index=0))


@pytest.mark.parametrize("call, message", [
    (lambda: kernels.expert_sort(Stub(4, 2), Stub(9, dtype=I32), SLOTS), "int32 or int64"),
    (lambda: kernels.expert_sort(Stub(8, dtype=I32), Stub(9, dtype=I32), SLOTS), "tokens x choices"),
    (lambda: kernels.expert_sort(Stub(4, 2, dtype=I32), Stub(1, dtype=I32), SLOTS), "one more value"),
    (lambda: kernels.expert_sort(Stub(4, 2, dtype=I32), Stub(9), SLOTS), "offsets must be"),
    (lambda: kernels.expert_sort(Stub(4, 3, dtype=I32), Stub(9, dtype=I32), SLOTS), "slots must be 4 x 3"),
    (lambda: kernels.expert_sort(Stub(4, 2, dtype=I32), Stub(9, dtype=I32), Stub(4, 2, dtype=torch.int64)), "in int32"),
    (lambda: kernels.expert_dispatch(Stub(5, 64), SLOTS, ROWS), "slots must be 5 x choices"),
    (lambda: kernels.expert_dispatch(X, SLOTS, Stub(8, 32)), "equally wide"),
    (lambda: kernels.expert_dispatch(X, SLOTS, Stub(8, 64, dtype=torch.float16)), "share one dtype"),
    (lambda: kernels.expert_dispatch(X, SLOTS, ROWS, weights=Stub(4, 3)), "weights must be"),
    (lambda: kernels.expert_dispatch(X, SLOTS, Stub(8, 64, device=0)), "share one device"),
    (lambda: kernels.expert_combine(Stub(8), SLOTS, X), "2-D"),
    (lambda: kernels.expert_combine_grad(X, ROWS, SLOTS, W, Stub(7, 64), W), "grad_y must be"),
    (lambda: kernels.expert_combine_grad(X, ROWS, SLOTS, W, ROWS, Stub(4, 2)), "grad_weights must be"),
    (lambda: kernels.quantize_fp4(X, Q, SCALES), "q must be"),
    (lambda: kernels.quantize_fp4(Stub(8, 96), Q, SCALES), "q must be"),
    (lambda: kernels.quantize_fp4(ROWS, Stub(8, 32), SCALES), "uint8"),
    (lambda: kernels.quantize_fp4(ROWS, Q, Stub(8, 2, dtype=U8)), "scales of q must be"),
    (lambda: kernels.quantize_fp4(Stub(8, 64, 1), Q, SCALES), "2-D"),
    (lambda: kernels.quantize_fp4(Stub(8, 48), Stub(8, 24, dtype=U8), SCALES), "multiple of 32"),
    (lambda: kernels.quantize_fp4(ROWS, Q, SCALES, slots=SLOTS), "slots must be 8"),
    (lambda: kernels.dequantize_fp4(Q, SCALES, X), "out must be"),
    (lambda: kernels.gemm_fp4(Q, SCALES, Stub(5, 16, dtype=U8), Stub(5, 16, dtype=U8), Stub(8, 5)), "incompatible"),
    (lambda: kernels.gemm_fp4(Q, SCALES, Stub(5, 32, dtype=U8), Stub(5, 32, dtype=U8), Stub(8, 5)), "scales of b"),
    (lambda: kernels.gemm_fp4(Q, SCALES, Stub(5, 32, dtype=U8), Stub(5, 16, dtype=U8), Stub(8, 6)), "out must be"),
    (lambda: kernels.gemm_fp4(Q, SCALES, Stub(2, 5, 32, dtype=U8), Stub(2, 5, 16, dtype=U8), Stub(8, 5)), "need offsets"),
])
def test_front_ends_refuse(machine, call, message):
    with pytest.raises(ValueError, match=message):
        call()
    assert not machine.launched


def test_scale_pitch():
    assert [kernels.fp4_scale_pitch(k) for k in (32, 512, 544, 4096, 16384)] == [16, 16, 32, 128, 512]


A = [P + 2 ** 24 * i for i in range(7)]  # far from each other, and never read


@pytest.mark.parametrize("entry, sizes, spans, written", [
    ("trb_expert_sort_launch", (4, 64, 8, 16), [64 * 8 * 4, 17 * 4, 64 * 8 * 4], (1, 2)),
    ("trb_expert_sort_launch", (8, 64, 8, 16), [64 * 8 * 8, 17 * 4, 64 * 8 * 4], (1, 2)),
    ("trb_expert_dispatch_launch", (BF16, F32, 16, 2, 32, 24), [16 * 48, 16 * 8, 16 * 8, 32 * 48], (3,)),
    ("trb_expert_combine_launch", (F32, F32, 16, 2, 32, 24), [32 * 96, 16 * 8, 16 * 8, 16 * 96], (3,)),
    ("trb_expert_combine_grad_launch", (BF16, BF16, 16, 2, 32, 24),
     [16 * 48, 32 * 48, 16 * 8, 16 * 4, 32 * 48, 16 * 4], (4, 5)),
    ("trb_dequantize_fp4_launch", (F16, 16, 64), [16 * 32, 16 * 16, 16 * 128], (2,)),
    ("trb_gemm_fp4_launch", (BF16, 4, 16, 24, 64), [16 * 32, 16 * 16, 4 * 24 * 32, 4 * 24 * 16, 5 * 4, 16 * 48], (5,)),
])
def test_results_that_overlap(entry, sizes, spans, written):
    """The same memory, its first bytes and its last ones, for each result and every other tensor."""
    for w in written:
        for other in range(len(spans)):
            for back in {0, 16, spans[other] // 16 * 16 - 16 if spans[other] % 16 == 0 else 0}:
                if other == w or back >= spans[other]:
                    continue
                if entry == "trb_expert_combine_grad_launch" and (w, other, back) == (4, 1, 0):
                    continue  # grad_y may be y itself
                at = A[:len(spans)]
                at[w] = at[other] + back
                assert getattr(_native.load(), entry)(*sizes, *at, None) == -1, (w, other, back)
                assert "must not overlap" in _native.last_error()


@pytest.mark.parametrize("slots, rows", [(None, 16), (P + 2 ** 20, 32)])
def test_quantised_results_that_overlap(slots, rows):
    x, q, scales = A[1:4]
    for over in ((x, x, scales), (x, x + 16 * 128 - 16, scales), (x, q, x), (x, q, q), (x, q, q + rows * 32 - 16),
                 *(((x, slots, scales), (x, q, slots)) if slots else ())):
        assert _native.load().trb_quantize_fp4_launch(BF16, 16, 64, over[0], 2, slots, rows, over[1], over[2], None) == -1
        assert "must not overlap" in _native.last_error()
