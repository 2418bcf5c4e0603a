"""Host side of the expert-layer products: the `experts` benchmark's registration, shares of rows and skipping, the
C entry points' refusals and the front ends' checks that need no GPU."""
from __future__ import annotations

import ctypes
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200 import builtin  # noqa: E402,F401
from teamredbench_b200.benchmarks.base import BenchmarkContext  # noqa: E402
from teamredbench_b200.benchmarks.experts import ExpertsBenchmark, expert_counts  # noqa: E402
from teamredbench_b200.config import HardwareProfile, RuntimeProfile, load_suite  # noqa: E402
from teamredbench_b200.dtypes import discover_dtypes  # noqa: E402
from teamredbench_b200.kernels import gemv_w4, grouped_gemm, grouped_gemm_wgrad  # noqa: E402
from teamredbench_b200.registry import list_benchmarks  # noqa: E402

SUITES = Path(__file__).resolve().parent.parent / "teamredbench_b200" / "configs" / "suites"
BF16, F32 = 1, 0


def test_registered_and_suite_loads():
    assert "experts" in list_benchmarks()
    suite = load_suite(SUITES / "b200_experts.yaml")
    assert {b.benchmark for b in suite.benchmarks} == {"experts"}
    for b in suite.benchmarks:
        for rows, experts, k, n in b.params["shapes"]:
            assert rows >= 1 and experts >= 1 and k % 8 == 0 and n % 8 == 0


@pytest.mark.parametrize("rows, experts, skew", [(0, 4, 0.5), (1, 8, 0.0), (1000, 16, 1.0)])
def test_counts_add_up_and_repeat(rows, experts, skew):
    counts = expert_counts(torch, rows, experts, skew, 3)
    assert counts.shape == (experts,) and int(counts.sum()) == rows and int(counts.min()) >= 0
    assert torch.equal(counts, expert_counts(torch, rows, experts, skew, 3))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the run without a GPU")
def test_without_a_gpu_the_benchmark_is_skipped():
    context = BenchmarkContext(hardware_profile=HardwareProfile(name="t", family="t"),
                               runtime_profile=RuntimeProfile(name="t"), device_info=None, torch_module=torch,
                               dtype_specs=discover_dtypes(torch))
    records = ExpertsBenchmark(context, {}).run()
    assert [r.status for r in records] == ["skipped"]


def test_front_ends_reject_host_tensors_before_launching():
    a, b = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16)
    offsets = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        grouped_gemm(a, b, offsets, torch.zeros_like(a))
    with pytest.raises(ValueError, match="CUDA device"):
        grouped_gemm_wgrad(a, a, offsets, b)
    with pytest.raises(ValueError, match="CUDA device"):
        gemv_w4(torch.zeros(1, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1), torch.zeros(1, 8))


P = 4096  # an aligned address that is never read: every call below is refused first


@pytest.mark.parametrize("args, status, message", [
    ((BF16, 0, 4, 8, 8, P, P, 0, P, P, None), -1, "sizes must be positive"),
    ((BF16, 1, -1, 8, 8, P, P, 0, P, P, None), -1, "sizes must be positive"),
    ((BF16, 1, 4, 8, 8, None, P, 0, P, P, None), -1, "non-null"),
    ((BF16, 1, 4, 8, 8, P, P, 0, None, P, None), -1, "non-null"),
    ((F32, 1, 4, 8, 8, P, P, 0, P, P, None), 1, "unsupported dtype"),
    ((BF16, 1025, 4, 8, 8, P, P, 0, P, P, None), 1, "at most 1024 groups"),
    ((BF16, 1, 4, 12, 8, P, P, 0, P, P, None), -3, "multiples of 8"),
    ((BF16, 1, 4, 8, 8, P + 2, P, 0, P, P, None), -3, "16-byte aligned"),
    ((BF16, 1, 4, 8, 8, P, P, 0, P + 2, P, None), -3, "4-byte aligned"),
    ((BF16, 1, 4, 8, 8, P, P, 7, P, P, None), -1, "unknown b_layout"),
    ((BF16, 1, 0, 8, 8, None, P, 0, P, None, None), 0, ""),
])
def test_grouped_gemm_entry(args, status, message):
    assert _native.load().trb_grouped_gemm_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("args, status, message", [
    ((BF16, 1, 4, 8, 8, P, P, P, None, None), -1, "non-null"),
    ((BF16, 1, 0, 8, 8, None, None, P, None, None), -1, "out is null"),
    ((BF16, 1, 4, 8, 0, P, P, P, P, None), -1, "sizes must be positive"),
    ((BF16, 1, 4, 8, 20, P, P, P, P, None), -3, "multiples of 8"),
    ((F32, 1, 4, 8, 8, P, P, P, P, None), 1, "unsupported dtype"),
])
def test_grouped_wgrad_entry(args, status, message):
    assert _native.load().trb_grouped_wgrad_launch(*args) == status
    assert message in _native.last_error()


@pytest.mark.parametrize("args, status, message", [
    ((BF16, 1, 1, 0, 64, 32, P, P, P, None, None, P, None), -1, "sizes must be positive"),
    ((BF16, 2, 1, 8, 64, 32, P, P, P, None, None, P, None), -1, "several groups need offsets"),
    ((BF16, 1, 1, 8, 64, 32, P, None, P, None, None, P, None), -1, "non-null"),
    ((F32, 1, 1, 8, 64, 32, P, P, P, None, None, P, None), 1, "unsupported dtype"),
    ((BF16, 1, 1, 8, 64, 16, P, P, P, None, None, P, None), 1, "group size"),
    ((BF16, 1, 1, 8, 96, 64, P, P, P, None, None, P, None), 1, "group size"),
    ((BF16, 1, 1, 8, 65536 + 32, 32, P, P, P, None, None, P, None), 1, "at most 65536"),
    ((BF16, 1, 1, 8, 64, 32, P + 8, P, P, None, None, P, None), -3, "16-byte aligned"),
    ((BF16, 1, 0, 8, 64, 32, None, P, P, None, None, None, None), 0, ""),
])
def test_gemv_w4_entry(args, status, message):
    assert _native.load().trb_gemv_w4_launch(*args) == status
    assert message in _native.last_error()


def test_header_and_binding_agree_on_the_number_of_arguments():
    lib = _native.load()
    assert len(lib.trb_grouped_gemm_launch.argtypes) == 11
    assert len(lib.trb_grouped_wgrad_launch.argtypes) == 10
    assert len(lib.trb_gemv_w4_launch.argtypes) == 13
    assert lib.trb_gemv_w4_launch.restype is ctypes.c_int
