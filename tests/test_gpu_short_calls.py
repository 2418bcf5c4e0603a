"""The compiled way from tensors to the library and the front ends' own: the same results, and the same refusals."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native, kernels  # noqa: E402

I32, U8, BF16 = torch.int32, torch.uint8, torch.bfloat16


def _make(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=BF16):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    t = {"ids": torch.randint(-1, 4, (9, 2), generator=g, device="cuda"), "offsets": torch.zeros(5, device="cuda", dtype=I32),
         "slots": torch.zeros(9, 2, device="cuda", dtype=I32), "x": randn(9, 64), "rows": torch.zeros(18, 64, device="cuda", dtype=BF16),
         "w": randn(9, 2, dtype=torch.float32), "y": randn(18, 64), "out": torch.zeros(9, 64, device="cuda", dtype=BF16),
         "grad_y": torch.zeros(18, 64, device="cuda", dtype=BF16), "grad_w": torch.zeros(9, 2, device="cuda"),
         "q": torch.zeros(18, 32, device="cuda", dtype=U8), "scales": torch.zeros(18, 16, device="cuda", dtype=U8),
         "values": torch.zeros(18, 64, device="cuda"), "product": torch.zeros(18, 40, device="cuda", dtype=torch.float16)}
    t["b"] = torch.randint(0, 256, (4, 40, 32), generator=g, device="cuda", dtype=U8)
    t["b_scales"] = torch.randint(120, 130, (4, 40, 16), generator=g, device="cuda", dtype=U8)
    return t


def _run(t):
    kernels.expert_sort(t["ids"], t["offsets"], t["slots"])
    kernels.expert_dispatch(t["x"], t["slots"], t["rows"], weights=t["w"])
    kernels.expert_combine(t["y"], t["slots"], t["out"])
    kernels.expert_combine_grad(t["out"], t["y"], t["slots"], t["w"], t["grad_y"], t["grad_w"])
    kernels.quantize_fp4(t["x"], t["q"], t["scales"], slots=t["slots"])
    kernels.dequantize_fp4(t["q"], t["scales"], t["values"])
    kernels.gemm_fp4(t["q"], t["scales"], t["b"], t["b_scales"], t["product"], offsets=t["offsets"])
    return t


def test_the_compiled_way_is_built_and_gives_the_same(monkeypatch):
    assert kernels._find_short(), "lib/trb_torch.so is missing or for another torch"
    short = _run(_make())
    monkeypatch.setattr(kernels, "_SHORT", False)
    long = _run(_make())
    for name in short:
        assert torch.equal(short[name], long[name]), name
    assert short["product"].any() and short["grad_w"].any()


def test_both_ways_are_taken(monkeypatch):
    """The front ends' own way is left alone where the compiled one did the call, and takes an explicit stream."""
    launched = []
    real = _native.expert_combine_launch
    monkeypatch.setattr(_native, "expert_combine_launch", lambda *a: (launched.append(a), real(*a)))
    t = _make()
    kernels.expert_sort(t["ids"], t["offsets"], t["slots"])
    kernels.expert_combine(t["y"], t["slots"], t["out"])
    assert not launched
    kernels.expert_combine(t["y"], t["slots"], t["out"], stream=torch.cuda.current_stream())
    assert len(launched) == 1


def test_takes_the_current_stream():
    t = _make()
    stream = torch.cuda.Stream()
    kernels.expert_sort(t["ids"], t["offsets"], t["slots"])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        kernels.expert_dispatch(t["x"], t["slots"], t["rows"])
        graph.capture_end()
    torch.cuda.synchronize()
    assert not t["rows"].any()  # captured on the stream that is current, not run
    graph.replay()
    torch.cuda.synchronize()
    assert t["rows"].any()


@pytest.mark.parametrize("name, value, message", [
    ("ids", lambda t: t["ids"].float(), "int32 or int64"),
    ("offsets", lambda t: t["offsets"][:1], "one more value"),
    ("slots", lambda t: t["slots"].t().contiguous(), "slots must be"),
    ("x", lambda t: t["x"].double(), "share one dtype"),
    ("x", lambda t: t["x"].cpu(), "CUDA device"),
    ("x", lambda t: t["x"].t(), "contiguous"),
    ("w", lambda t: t["w"].half(), "weights must be"),
    ("out", lambda t: t["out"][:, :32].contiguous(), "equally wide"),
    ("grad_w", lambda t: t["grad_w"].bfloat16(), "grad_weights must be"),
    ("scales", lambda t: t["scales"][:, :8].contiguous(), "scales of q"),
    ("q", lambda t: t["q"].int(), "uint8"),
    ("values", lambda t: t["values"][:, :32].contiguous(), "out must be"),
    ("b", lambda t: t["b"][:3].contiguous(), "scales of b|need|offsets must"),
    ("product", lambda t: t["product"].float(), "unsupported dtype"),
])
def test_what_is_wrong_is_named(name, value, message):
    t = _make()
    t[name] = value(t)
    with pytest.raises((ValueError, _native.NativeError), match=message):
        _run(t)
    torch.cuda.synchronize()


@pytest.mark.parametrize("k", [16, 48])
def test_a_size_that_the_library_refuses_is_an_error(k):
    t = _make()
    with pytest.raises(ValueError, match="multiple of 32"):
        kernels.quantize_fp4(t["x"][:, :k].contiguous(), torch.zeros(9, k // 2, device="cuda", dtype=U8),
                             torch.zeros(9, 16, device="cuda", dtype=U8))
