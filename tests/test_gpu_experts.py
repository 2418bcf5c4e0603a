"""The `experts` benchmark on the GPU: forward, training step and 4-bit decode of one expert layer through a suite."""
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


def test_suite_runs_every_mode(tmp_path):
    suite = tmp_path / "suite.yaml"
    suite.write_text(yaml.safe_dump({
        "name": "experts", "device": {"profile": str(HW)}, "runtime": {"profile": str(RT)},
        "outputs": {"directory": str(tmp_path / "results"), "formats": ["json", "csv"]},
        "benchmarks": [{"benchmark": "experts", "params": {
            "dtypes": ["bfloat16", "float16", "float32"], "modes": ["forward", "train", "decode_w4"],
            "shapes": [[300, 8, 1024, 512], [5, 8, 1024, 512]], "group": 64, "warmup": 1, "iterations": 3}}]}),
        encoding="utf-8")
    summary = run_suite(suite)
    by_key = {(r.case, r.dtype): r for r in summary.records}
    for rows in (300, 5):
        for mode in ("forward", "train", "decode_w4"):
            case = f"{mode}_{rows}x8x1024x512"
            for dtype in ("bfloat16", "float16"):
                r = by_key[(case, dtype)]
                assert r.status == "ok", r.error
                assert r.metadata["device_error"] == 0
                assert r.metrics["achieved_tops"] > 0 and r.metrics["hbm_bandwidth_gbps"] > 0
                factor = 3 if mode == "train" else 1
                assert r.raw_metrics["achieved_ops"] == factor * 2 * rows * 1024 * 512
            assert by_key[(case, "float32")].status == "skipped"
