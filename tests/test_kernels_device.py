"""The torch front ends launch on the device that their tensors are on, whichever is current (two devices played by
stub tensors and a recording library: no GPU)."""
from __future__ import annotations

import contextlib
import types

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200 import _native, kernels  # noqa: E402


class Stub:
    """What the front ends ask of a tensor, on device 1."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.bfloat16, device=1):
        self.shape, self.dtype, self.index = torch.Size(shape), dtype, device
        self.device = f"cuda:{device}"

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def data_ptr(self):
        return 4096


OFFSETS = Stub(3, dtype=torch.int32)
CALLS = {
    "grouped_gemm_launch": lambda **kw: kernels.grouped_gemm(Stub(4, 8), Stub(2, 8, 16), OFFSETS, Stub(4, 16), **kw),
    "grouped_wgrad_launch": lambda **kw: kernels.grouped_gemm_wgrad(Stub(4, 8), Stub(4, 16), OFFSETS, Stub(2, 8, 16),
                                                                    **kw),
    "gemv_w4_launch": lambda **kw: kernels.gemv_w4(Stub(4, 64), Stub(8, 32, dtype=torch.uint8), Stub(8, 1),
                                                   Stub(4, 8), **kw),
    "gemm_launch_ex": lambda **kw: kernels.gemm(Stub(4, 8), Stub(8, 16), Stub(4, 16), **kw),
    "hbm_launch": lambda **kw: kernels.stream_op("copy", Stub(64), Stub(64), **kw),
}


@pytest.fixture
def machine(monkeypatch):
    """Two devices; `current` is the thread's, `entered` counts the switches, `launched` holds one device a launch."""
    m = types.SimpleNamespace(current=0, entered=0, launched=[], fail=False)

    @contextlib.contextmanager
    def device(index):
        before, m.current = m.current, index
        m.entered += 1
        try:
            yield
        finally:
            m.current = before

    def launch(*args, **kw):
        m.launched.append(m.current)
        if m.fail:
            raise _native.NativeError(-2, "refused")

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(kernels, "_CURRENT_DEVICE", lambda: m.current, raising=False)
    monkeypatch.setattr(kernels, "_RAW_STREAM", lambda index: 0)  # every device's default stream is 0
    for name in CALLS:
        monkeypatch.setattr(_native, name, launch)
    return m


@pytest.mark.parametrize("call", CALLS)
def test_launches_on_the_tensors_device(machine, call):
    CALLS[call]()
    assert machine.launched == [1] and machine.current == 0


@pytest.mark.parametrize("call", CALLS)
def test_the_current_device_comes_back_after_an_error(machine, call):
    machine.fail = True
    with pytest.raises(_native.NativeError):
        CALLS[call]()
    assert machine.launched == [1] and machine.current == 0


@pytest.mark.parametrize("call", CALLS)
def test_nothing_is_switched_where_the_device_is_current(machine, call):
    machine.current = 1
    CALLS[call]()
    assert machine.launched == [1] and machine.entered == 0


@pytest.mark.parametrize("call", CALLS)
def test_a_stream_of_another_device_is_refused(machine, call):
    with pytest.raises(ValueError, match="stream is on cuda:0"):
        CALLS[call](stream=types.SimpleNamespace(cuda_stream=0, device_index=0))
    CALLS[call](stream=types.SimpleNamespace(cuda_stream=77, device_index=1))
    assert machine.launched == [1]
