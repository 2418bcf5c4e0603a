"""The `experts` benchmark's whole-layer modes without a GPU: the tokens' choices, the calls of a step, their operations."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200.benchmarks import experts  # noqa: E402
from tests.test_experts_records import bench  # noqa: E402,F401

CALLS = ("expert_sort", "expert_dispatch", "expert_combine", "expert_combine_grad", "quantize_fp4", "gemm_fp4")


@pytest.mark.parametrize("counts, choices", [([3, 0, 5], 1), ([3, 0, 5], 3), ([0, 0], 2), ([1], 4), ([40, 2, 0, 21], 2)])
def test_choices_are_the_counts_dealt_out_to_tokens(counts, choices):
    counts = torch.tensor(counts)
    ids = experts.expert_choices(torch, counts, choices, 1)
    rows = int(counts.sum())
    assert ids.shape == (-(-rows // choices), choices) and ids.dtype is torch.int64
    assert torch.equal(torch.bincount(ids[ids >= 0], minlength=counts.numel()), counts)
    assert int((ids < 0).sum()) == ids.numel() - rows
    assert torch.equal(ids, experts.expert_choices(torch, counts, choices, 1))


@pytest.mark.parametrize("mode, want", [
    ("layer", ["expert_sort", "expert_dispatch", "grouped_gemm", "expert_combine"]),
    ("layer_train", ["expert_sort", "expert_dispatch", "grouped_gemm", "expert_combine", "expert_combine_grad",
                     "grouped_gemm", "grouped_gemm_wgrad", "expert_combine"]),
    ("layer_fp4", ["expert_sort", "quantize_fp4", "gemm_fp4", "expert_combine"]),
])
def test_a_step_is_these_calls(bench, monkeypatch, mode, want):  # noqa: F811
    calls = []
    for name in CALLS + ("grouped_gemm", "grouped_gemm_wgrad"):
        monkeypatch.setattr(experts, name, lambda *a, _name=name, **k: calls.append((_name, a)))
    bench.l2 = 10  # one set of operands
    (record,) = bench.run(mode)
    assert record.status == "ok" and record.metadata["choices"] == 2
    factor = 3 if mode == "layer_train" else 1
    assert record.raw_metrics["achieved_ops"] == factor * 2 * 8 * 64 * 64 and record.raw_metrics["moved_bytes"] > 0
    steps = [name for name, _ in calls]
    first = steps.index("expert_sort")
    assert steps[first:first + len(want)] == want
    # What one call writes the next one reads.
    args = [a for _, a in calls[first:first + len(want)]]
    assert args[0][2] is (args[1][1] if mode != "layer_fp4" else args[3][1])  # slots


def test_the_layers_are_not_among_the_default_modes(bench):  # noqa: F811
    assert experts.DEFAULT_MODES == ("forward", "train", "decode_w4")
    with pytest.raises(KeyError, match="layers"):
        bench.run("layers")
