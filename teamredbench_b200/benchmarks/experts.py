"""Matrix products of an expert (mixture-of-experts) layer, and the layer around them, in process through
libtrb_b200 (no reference counterpart; records, metrics and skipping follow
src/teamredbench/benchmarks/mfu.py).

One case per (mode, shape) with shape [rows, experts, k, n]: `rows` rows are
dealt out to the experts unevenly (`skew`, 0 = evenly on average) and sorted by
expert.
  forward    out = rows x (k x n) weights of their expert
  train      forward, then the gradients of the rows and of the weights
  decode_w4  the forward product with 4-bit weights, a scale and a zero point
             per `group` k
  layer      the rows are the choices of tokens, `choices` each: sorted by
             expert, the tokens' rows dispatched, the forward product, and the
             results combined with the router's weights
  layer_train  layer, then all its gradients: of the experts' rows and the
             router's weights, of the dispatched rows and the matrices, and of
             the tokens' rows
  layer_fp4  layer in microscaled 4-bit floating point: the tokens are
             quantised into their experts' rows, against quantised matrices; its
             MFU is of the hardware profile's float4_e2m1 peak
The first three are the default.

The calls of a case take several sets of operands in turn, which together move
three times what the L2 holds, so that the bytes come from the memory whose
bandwidth is reported; where so many sets do not fit, no moved bytes are
recorded.  Time is a host loop's: calls of a few microseconds show the host.
"""
from __future__ import annotations

import itertools
from typing import Any

from teamredbench_b200 import _native
from teamredbench_b200.benchmarks.base import Benchmark, BenchmarkRecord
from teamredbench_b200.device import cuda_device_available
from teamredbench_b200.kernels import (expert_combine, expert_combine_grad, expert_dispatch, expert_sort,
                                        fp4_scale_pitch, gemm_fp4, gemv_w4, grouped_gemm, grouped_gemm_wgrad,
                                        quantize_fp4)
from teamredbench_b200.registry import register_benchmark
from teamredbench_b200.utils import timed_iterations

DEFAULT_MODES = ("forward", "train", "decode_w4")
LAYER_MODES = ("layer", "layer_train", "layer_fp4")
MODES = DEFAULT_MODES + LAYER_MODES
DTYPES = ("bfloat16", "float16")


def expert_counts(torch_module: Any, rows: int, experts: int, skew: float, seed: int):
    """Rows of each expert, on the host: shares proportional to exp(skew * N(0, 1))."""
    torch = torch_module
    gen = torch.Generator().manual_seed(seed)
    share = torch.exp(skew * torch.randn(experts, generator=gen, dtype=torch.float64))
    if rows == 0:
        return torch.zeros(experts, dtype=torch.int64)
    return torch.bincount(torch.multinomial(share, rows, replacement=True, generator=gen), minlength=experts)


def expert_choices(torch_module: Any, counts: Any, choices: int, seed: int):
    """The experts (tokens x choices, int64) of as many tokens as the rows take, each expert as often as `counts` says,
    in any order; -1 where the last token has fewer choices."""
    torch = torch_module
    rows = int(counts.sum())
    tokens = -(-rows // choices)
    ids = torch.full((tokens * choices,), -1, dtype=torch.int64)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(seed))
    ids[:rows] = torch.repeat_interleave(torch.arange(counts.numel()), counts)[order]
    return ids.view(tokens, choices)


def operand_sets(moved: int, held: int, l2_bytes: int, free_bytes: int) -> tuple[int, bool]:
    """(sets of operands to use in turn, whether none is still in L2 when its turn comes) for calls that move `moved`
    of the `held` bytes of a set: what three times the L2 takes, as far as it fits in half the free memory."""
    want = -(-3 * l2_bytes // moved) if moved else 1
    sets = max(1, min(want, 512, 1 + free_bytes // 2 // held))
    return sets, sets >= want


def device_memory(torch_module: Any, device: Any) -> tuple[int, int]:
    """(bytes of L2, bytes of free memory) of a CUDA device."""
    l2 = getattr(torch_module.cuda.get_device_properties(device), "L2_cache_size", 128 << 20)
    return l2, torch_module.cuda.mem_get_info(device)[0]


@register_benchmark("experts")
class ExpertsBenchmark(Benchmark):
    default_metrics = ["achieved_tops", "mfu_pct", "hbm_bandwidth_gbps", "latency_us"]

    def _step(self, mode: str, dtype: Any, counts: Any, k: int, n: int, group: int, gen: Any):
        """(the call of one step, its multiply-add operations, its algorithmic bytes, the bytes of its operands)."""
        torch, dev = self.torch, self.device
        rows, experts = int(counts.sum()), counts.numel()
        active = int((counts > 0).sum())
        offsets = torch.zeros(experts + 1, dtype=torch.int32)
        offsets[1:] = torch.cumsum(counts, 0)
        offsets = offsets.to(dev)
        flops, row_bytes, weight_bytes = 2 * rows * k * n, 2 * rows * (k + n), 2 * k * n

        def held(*tensors):
            return sum(t.numel() * t.element_size() for t in tensors)

        def randn(*shape, scale=1.0):
            return (torch.randn(shape, device=dev, generator=gen) * scale).to(dtype)

        if mode in LAYER_MODES:
            return self._layer(mode, dtype, counts, k, n, randn, held)
        a, out = randn(rows, k), torch.empty((rows, n), device=dev, dtype=dtype)
        if mode == "decode_w4":
            q = torch.randint(0, 256, (experts, n, k // 2), device=dev, dtype=torch.uint8, generator=gen)
            scales = randn(experts, n, k // group, scale=k ** -0.5 / 4.6)
            zeros = torch.randint(0, 16, scales.shape, device=dev, dtype=torch.uint8, generator=gen)
            return (lambda: gemv_w4(a, q, scales, out, zeros=zeros, offsets=offsets), flops,
                    row_bytes + active * (n * k // 2 + 3 * n * (k // group)), held(a, out, q, scales, zeros))
        b = randn(experts, k, n, scale=k ** -0.5)
        if mode == "forward":
            return (lambda: grouped_gemm(a, b, offsets, out), flops, row_bytes + active * weight_bytes,
                    held(a, out, b))
        grad, grad_a, grad_b = randn(rows, n), torch.empty_like(a), torch.empty_like(b)

        def train() -> None:
            grouped_gemm(a, b, offsets, out)
            grouped_gemm(grad, b, offsets, grad_a, b_transposed=True)
            grouped_gemm_wgrad(a, grad, offsets, grad_b)

        return (train, 3 * flops, 3 * row_bytes + (2 * active + experts) * weight_bytes,
                held(a, out, b, grad, grad_a, grad_b))

    def _layer(self, mode: str, dtype: Any, counts: Any, k: int, n: int, randn: Any, held: Any):
        """_step for the whole layer."""
        torch, dev = self.torch, self.device
        rows, experts = int(counts.sum()), counts.numel()
        active = int((counts > 0).sum())
        ids = expert_choices(torch, counts, int(self.params.get("choices", 2)), int(self.params.get("seed", 0))).to(dev)
        tokens = ids.shape[0]

        def empty(*shape, dtype=dtype):
            return torch.empty(shape, device=dev, dtype=dtype)

        offsets, slots = empty(experts + 1, dtype=torch.int32), empty(*ids.shape, dtype=torch.int32)
        weights = torch.softmax(randn(*ids.shape).float(), 1)
        x, y, out = randn(tokens, k), empty(rows, n), empty(tokens, n)
        plan = held(ids, slots, weights) + held(slots)  # written, then read
        flops, moved = 2 * rows * k * n, plan + 2 * (tokens * k + tokens * n + 2 * rows * n)
        if mode == "layer_fp4":
            block = k // 2 + k // 32  # codes and scales of a row
            a, a_scales = empty(rows, k // 2, dtype=torch.uint8), empty(rows, fp4_scale_pitch(k), dtype=torch.uint8)
            b, b_scales = empty(experts, n, k // 2, dtype=torch.uint8), empty(experts, n, fp4_scale_pitch(k),
                                                                              dtype=torch.uint8)
            for e in range(experts):
                quantize_fp4(randn(n, k, scale=k ** -0.5), b[e], b_scales[e])

            def layer_fp4() -> None:
                expert_sort(ids, offsets, slots)
                quantize_fp4(x, a, a_scales, slots=slots)
                gemm_fp4(a, a_scales, b, b_scales, y, offsets=offsets)
                expert_combine(y, slots, out, weights=weights)

            return layer_fp4, flops, moved + 2 * rows * block + active * n * block, held(x, y, out, a, a_scales, b, b_scales)
        xs, b = empty(rows, k), randn(experts, k, n, scale=k ** -0.5)

        def layer() -> None:
            expert_sort(ids, offsets, slots)
            expert_dispatch(x, slots, xs)
            grouped_gemm(xs, b, offsets, y)
            expert_combine(y, slots, out, weights=weights)

        moved += 4 * rows * k + 2 * active * k * n
        if mode == "layer":
            return layer, flops, moved, held(x, y, out, xs, b)
        grad, grad_y, grad_weights = randn(tokens, n), empty(rows, n), torch.empty_like(weights)
        grad_xs, grad_x, grad_b = empty(rows, k), empty(tokens, k), torch.empty_like(b)

        def layer_train() -> None:
            layer()
            expert_combine_grad(grad, y, slots, weights, grad_y, grad_weights)
            grouped_gemm(grad_y, b, offsets, grad_xs, b_transposed=True)
            grouped_gemm_wgrad(xs, grad_y, offsets, grad_b)
            expert_combine(grad_xs, slots, grad_x)

        moved += (held(slots, weights, grad_weights, slots) + 2 * (tokens * n + 4 * rows * n)
                  + 2 * (3 * rows * k + tokens * k) + 2 * (active + experts) * k * n)
        return (layer_train, 3 * flops, moved,
                held(x, y, out, xs, b, grad, grad_y, grad_weights, grad_xs, grad_x, grad_b))

    def _measure(self, metadata: dict[str, Any], mode: str, dtype: Any, counts: Any, k: int, n: int,
                 group: int) -> dict[str, Any]:
        """Time, operations and bytes of one case's call; its operands are gone when this returns."""
        p = self.params
        gen = self.torch.Generator(device=self.device).manual_seed(int(p.get("seed", 0)))
        step, ops, moved, held = self._step(mode, dtype, counts, k, n, group, gen)
        sets, cold = operand_sets(moved, held, *device_memory(self.torch, self.device))
        metadata["operand_sets"] = sets
        turn = itertools.cycle([step] + [self._step(mode, dtype, counts, k, n, group, gen)[0] for _ in range(sets - 1)])
        _native.device_error(self.context.device_id, clear=True)  # of earlier calls
        self.sync_ranks()
        elapsed_s = timed_iterations(lambda: next(turn)(), torch_module=self.torch, warmup=int(p.get("warmup", 10)),
                                     iterations=int(p.get("iterations", 50)))
        code = metadata["device_error"] = _native.device_error(self.context.device_id, clear=True)
        if code:
            raise RuntimeError(f"the kernels set the device error word to {code}")
        return {"elapsed_s": elapsed_s, "achieved_ops": ops, "moved_bytes": moved if cold else None}

    def run(self) -> list[BenchmarkRecord]:
        p = self.params
        if self.context.torch_module is None:
            return [self.emit_record(self.skipped_record(case="global", dtype="n/a", error="PyTorch is not installed."))]
        torch = self.torch
        if not cuda_device_available(torch):
            return [self.emit_record(self.skipped_record(case="global", dtype="n/a",
                                                         error="No CUDA device visible to PyTorch."))]
        self.set_device()
        modes = list(p.get("modes", DEFAULT_MODES))
        for mode in modes:
            if mode not in MODES:
                raise KeyError(f"Unknown experts mode: {mode}")
        skew, seed, group = float(p.get("skew", 0.5)), int(p.get("seed", 0)), int(p.get("group", 128))
        profile = self.context.hardware_profile
        records: list[BenchmarkRecord] = []
        for spec in self.selected_dtype_specs():
            for rows, experts, k, n in ([int(d) for d in shape] for shape in p.get("shapes", [[4096, 16, 2048, 4096]])):
                counts = expert_counts(torch, rows, experts, skew, seed)
                for mode in modes:
                    case = f"{mode}_{rows}x{experts}x{k}x{n}"
                    metadata: dict[str, Any] = {"backend": "native", "backend_library": "libtrb_b200", "mode": mode,
                                                "rows": rows, "experts": experts, "k": k, "n": n, "skew": skew,
                                                "most_rows": int(counts.max())}
                    if mode == "decode_w4":
                        metadata["group"] = group
                    if mode in LAYER_MODES:
                        metadata["choices"] = int(p.get("choices", 2))
                    if spec.name not in DTYPES:
                        records.append(self.emit_record(self.skipped_record(
                            case=case, dtype=spec.name, error="The expert products take bfloat16 and float16.",
                            metadata=metadata)))
                        continue
                    try:
                        raw = self._measure(metadata, mode, getattr(torch, spec.torch_attr), counts, k, n, group)
                    except Exception as exc:  # noqa: BLE001 - any failure becomes a skipped record
                        records.append(self.emit_record(self.skipped_record(case=case, dtype=spec.name, error=str(exc),
                                                                            metadata=metadata)))
                        continue
                    records.append(self.emit_record(BenchmarkRecord(
                        benchmark=self.name, case=case, dtype=spec.name,
                        raw_metrics={**raw,
                                     "peak_tops": profile.peak_compute_tops.get(
                                         "float4_e2m1" if mode == "layer_fp4" else spec.name),
                                     "peak_bandwidth_gbps": profile.peak_hbm_bandwidth_gbps},
                        metadata=metadata)))
        return records
