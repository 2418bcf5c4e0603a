"""What one call of the `experts` benchmark's whole-layer modes writes the next one reads, without a GPU."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from teamredbench_b200.benchmarks import experts  # noqa: E402
from tests.test_experts_records import bench  # noqa: E402,F401

CALLS = ("expert_sort", "expert_dispatch", "expert_combine", "expert_combine_grad", "quantize_fp4", "gemm_fp4",
         "grouped_gemm", "grouped_gemm_wgrad")
LAYER = [
    "expert_sort ids offsets slots",
    "expert_dispatch x slots xs",
    "grouped_gemm xs b offsets y",
    "expert_combine y slots out weights=weights",
]
STEPS = {
    "layer": LAYER,
    "layer_train": LAYER + [
        "expert_combine_grad grad y slots weights grad_y grad_weights",
        "grouped_gemm grad_y b offsets grad_xs b_transposed=True",
        "grouped_gemm_wgrad xs grad_y offsets grad_b",
        "expert_combine grad_xs slots grad_x",
    ],
    "layer_fp4": [
        "expert_sort ids offsets slots",
        "quantize_fp4 x a a_scales slots=slots",
        "gemm_fp4 a a_scales b b_scales y offsets=offsets",
        "expert_combine y slots out weights=weights",
    ],
}
ROWS, EXPERTS, K, N = 8, 2, 64, 64  # the fixture's case, with two choices a token
SHAPES = {"ids": (4, 2), "slots": (4, 2), "weights": (4, 2), "grad_weights": (4, 2), "offsets": (EXPERTS + 1,),
          "x": (4, K), "grad_x": (4, K), "xs": (ROWS, K), "grad_xs": (ROWS, K), "y": (ROWS, N), "grad_y": (ROWS, N),
          "out": (4, N), "grad": (4, N), "a": (ROWS, K // 2), "a_scales": (ROWS, 16)}
MATRICES = {"layer": {"b": (EXPERTS, K, N)}, "layer_train": {"b": (EXPERTS, K, N), "grad_b": (EXPERTS, K, N)},
            "layer_fp4": {"b": (EXPERTS, N, K // 2), "b_scales": (EXPERTS, N, 16)}}


@pytest.mark.parametrize("mode", STEPS)
def test_what_one_call_writes_the_next_one_reads(bench, monkeypatch, mode):  # noqa: F811
    """A name is one tensor of the same shape in all calls of a step, and no two names are the same one."""
    calls = []
    for name in CALLS:
        monkeypatch.setattr(experts, name, lambda *a, _name=name, **k: calls.append((_name, a, k)))
    bench.l2 = 10  # one set of operands
    (record,) = bench.run(mode)
    assert record.status == "ok"
    names = [name for name, *_ in calls]
    first, want = names.index("expert_sort"), STEPS[mode]
    tensors = {}

    def same(name, tensor):
        assert tensors.setdefault(name, tensor) is tensor, name

    for line, (call, args, keywords) in zip(want, calls[first:first + len(want)], strict=True):
        words = line.split()
        positional = [word for word in words[1:] if "=" not in word]
        named = dict(word.split("=") for word in words[1:] if "=" in word)
        assert call == words[0] and len(args) == len(positional) and set(keywords) == set(named), line
        for name, tensor in zip(positional, args):
            same(name, tensor)
        for keyword, name in named.items():
            if name == "True":
                assert keywords[keyword] is True
            else:
                same(name, keywords[keyword])
    assert len({id(t) for t in tensors.values()}) == len({t.data_ptr() for t in tensors.values()}) == len(tensors)
    for name, tensor in tensors.items():
        assert tuple(tensor.shape) == {**SHAPES, **MATRICES[mode]}[name], name
    # The steps after it are the same calls again, on the same operands.
    later = calls[first + len(want):first + 2 * len(want)]
    assert [(c, [id(t) for t in a]) for c, a, _ in later] == [(c, [id(t) for t in a]) for c, a, _ in
                                                              calls[first:first + len(want)]]
