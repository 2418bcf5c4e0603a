"""What the `experts` benchmark records, with the library and the GPU replaced by stand-ins."""
from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200 import builtin  # noqa: E402,F401
from teamredbench_b200.benchmarks import experts  # noqa: E402
from teamredbench_b200.benchmarks.base import BenchmarkContext  # noqa: E402
from teamredbench_b200.config import HardwareProfile, RuntimeProfile  # noqa: E402
from teamredbench_b200.dtypes import discover_dtypes  # noqa: E402


@pytest.fixture
def bench(monkeypatch):
    """A benchmark of one case whose call sets the error word to `gpu.error` and takes `gpu.seconds`."""
    gpu = types.SimpleNamespace(word=0, error=0, seconds=1e-3)

    def device_error(device_id=0, clear=False):
        word = gpu.word
        if clear:
            gpu.word = 0
        return word

    def timed(fn, **_):
        gpu.word = gpu.word or gpu.error
        return gpu.seconds

    monkeypatch.setattr(experts, "cuda_device_available", lambda _: True)
    monkeypatch.setattr(experts, "timed_iterations", timed)
    monkeypatch.setattr(experts._native, "device_error", device_error)
    monkeypatch.setattr(experts.ExpertsBenchmark, "device", "cpu")
    monkeypatch.setattr(experts.ExpertsBenchmark, "set_device", lambda self: None)
    for product in ("grouped_gemm", "grouped_gemm_wgrad", "gemv_w4"):
        monkeypatch.setattr(experts, product, lambda *a, **k: None)
    context = BenchmarkContext(hardware_profile=HardwareProfile(name="t", family="t"),
                               runtime_profile=RuntimeProfile(name="t"), device_info=None, torch_module=torch,
                               dtype_specs=discover_dtypes(torch))
    gpu.run = lambda: experts.ExpertsBenchmark(context, {"dtypes": ["bfloat16"], "modes": ["forward"],
                                                         "shapes": [[8, 2, 64, 64]]}).run()
    return gpu


def test_a_clean_run_is_ok(bench):
    (record,) = bench.run()
    assert record.status == "ok" and record.metadata["device_error"] == 0
    assert record.raw_metrics["elapsed_s"] == bench.seconds


@pytest.mark.parametrize("code", [1, 3, 7])
def test_a_set_error_word_is_no_result(bench, code):
    """A call that gave up or refused its offsets computed little or nothing: its time is not a throughput."""
    bench.error = code
    (record,) = bench.run()
    assert record.status == "skipped" and str(code) in record.error
    assert record.metadata["device_error"] == code and not record.raw_metrics
    assert bench.word == 0


def test_an_older_error_is_not_charged_to_the_run(bench):
    bench.word = 2
    (record,) = bench.run()
    assert record.status == "ok" and record.metadata["device_error"] == 0
