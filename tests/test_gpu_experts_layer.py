"""The `experts` benchmark's whole-layer modes on the GPU, through a suite."""
from __future__ import annotations

from pathlib import Path

import pytest
import yaml

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200.runner import run_suite  # noqa: E402

ROOT = Path(__file__).resolve().parent.parent
HW = ROOT / "teamredbench_b200" / "configs" / "profiles" / "hardware" / "nvidia_b200.yaml"
RT = ROOT / "teamredbench_b200" / "configs" / "profiles" / "cuda" / "cuda_generic.yaml"


def test_suite_runs_the_layers(tmp_path):
    suite = tmp_path / "suite.yaml"
    suite.write_text(yaml.safe_dump({
        "name": "layers", "device": {"profile": str(HW)}, "runtime": {"profile": str(RT)},
        "outputs": {"directory": str(tmp_path / "results"), "formats": ["json"]},
        "benchmarks": [{"benchmark": "experts", "params": {
            "dtypes": ["bfloat16", "float16"], "modes": ["layer", "layer_train", "layer_fp4"],
            "shapes": [[301, 8, 1024, 512], [5, 8, 1024, 520]], "choices": 3, "warmup": 1, "iterations": 3}},
            {"benchmark": "experts", "params": {"dtypes": ["bfloat16"], "modes": ["layer_fp4"], "shapes": [[64, 4, 1000, 512]],
                                                "warmup": 1, "iterations": 1}}]}),
        encoding="utf-8")
    records = run_suite(suite).records
    by_key = {(r.case, r.dtype): r for r in records}
    for rows, n in ((301, 512), (5, 520)):
        for mode in ("layer", "layer_train", "layer_fp4"):
            for dtype in ("bfloat16", "float16"):
                r = by_key[(f"{mode}_{rows}x8x1024x{n}", dtype)]
                assert r.status == "ok", r.error
                assert r.metadata["device_error"] == 0 and r.metadata["choices"] == 3
                assert r.metrics["achieved_tops"] > 0 and r.metrics["hbm_bandwidth_gbps"] > 0
                assert r.raw_metrics["peak_tops"] == (9000.0 if mode == "layer_fp4" else 2250.0)
    refused = by_key[("layer_fp4_64x4x1000x512", "bfloat16")]  # k is no multiple of 32
    assert refused.status == "skipped" and "32" in refused.error
