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
    gpu = types.SimpleNamespace(word=0, error=0, seconds=1e-3, l2=20000, free=1 << 30, calls=[])

    def device_error(device_id=0, clear=False):
        word = gpu.word
        if clear:
            gpu.word = 0
        return word

    def timed(fn, **_):
        for _ in range(12):
            fn()
        gpu.word = gpu.word or gpu.error
        return gpu.seconds

    monkeypatch.setattr(experts, "cuda_device_available", lambda _: True)
    monkeypatch.setattr(experts, "timed_iterations", timed)
    monkeypatch.setattr(experts._native, "device_error", device_error)
    monkeypatch.setattr(experts, "device_memory", lambda torch_module, device: (gpu.l2, gpu.free), raising=False)
    monkeypatch.setattr(experts.ExpertsBenchmark, "device", "cpu")
    monkeypatch.setattr(experts.ExpertsBenchmark, "set_device", lambda self: None)
    for product in ("grouped_gemm", "grouped_gemm_wgrad", "gemv_w4"):
        monkeypatch.setattr(experts, product, lambda *a, **k: gpu.calls.append(a))
    context = BenchmarkContext(hardware_profile=HardwareProfile(name="t", family="t"),
                               runtime_profile=RuntimeProfile(name="t"), device_info=None, torch_module=torch,
                               dtype_specs=discover_dtypes(torch))
    gpu.run = lambda mode="forward": experts.ExpertsBenchmark(
        context, {"dtypes": ["bfloat16"], "modes": [mode], "shapes": [[8, 2, 64, 64]], "group": 32}).run()
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


@pytest.mark.parametrize("mode, calls", [("forward", 1), ("train", 3), ("decode_w4", 1)])
def test_operands_are_taken_in_turn_from_more_than_the_l2_holds(bench, mode, calls):
    """Operands that stay in L2 would give its bandwidth under the name of the memory's."""
    (record,) = bench.run(mode)
    sets = record.metadata["operand_sets"]
    assert sets > 1 and sets * record.raw_metrics["moved_bytes"] >= 3 * bench.l2
    weights = [c[1].data_ptr() for c in bench.calls[::calls]]
    rows = [c[0].data_ptr() for c in bench.calls[::calls]]
    for used in (weights, rows):
        assert len(set(used[:sets])) == sets and used[sets:2 * sets] == used[:min(sets, 12 - sets)]


def test_large_operands_need_one_set(bench):
    bench.l2 = 10
    (record,) = bench.run()
    assert record.metadata["operand_sets"] == 1 and record.raw_metrics["moved_bytes"] > 0


def test_no_bandwidth_where_the_sets_do_not_fit(bench):
    bench.free = 1
    (record,) = bench.run()
    assert record.status == "ok" and record.metadata["operand_sets"] == 1
    assert record.raw_metrics["moved_bytes"] is None and record.raw_metrics["achieved_ops"] > 0


@pytest.mark.parametrize("moved, held, l2, free, want", [
    (1000, 1000, 0, 10 ** 9, (1, True)), (10 ** 9, 10 ** 9, 126 << 20, 10 ** 11, (1, True)),
    (44 * 10 ** 6, 67 * 10 ** 6, 126 << 20, 10 ** 11, (10, True)),
    (33 * 10 ** 6, 34 * 10 ** 9, 126 << 20, 150 * 10 ** 9, (3, False)), (16, 16, 126 << 20, 10 ** 11, (512, False)),
    (0, 64, 126 << 20, 10 ** 11, (1, True)),
])
def test_operand_sets(moved, held, l2, free, want):
    assert experts.operand_sets(moved, held, l2, free) == want
