"""Workloads of the expert-layer operators: ragged grouped products, their weight gradient, 4-bit products.

Three operators of a mixture-of-experts feed-forward block, as a training or serving program calls them:

``grouped``  out[r] = a[r] @ b[e] for the rows r of expert e (forward, or the gradient of the rows with ``b_transposed``)
``wgrad``    out[e] = a[rows of e]^T @ grad[rows of e]
``w4``       out[r] = x[r] @ W[e]^T with W = (q - z) * s, q in 4 bits, one scale s (and zero point z) per group of k

Rows are sorted by expert; ``offsets`` (experts + 1 numbers on the device) says where each expert's rows begin.
"""
import math

import torch

own = False

MAX_MACS = 32768 * 4096 * 4096
MAX_WEIGHTS = 1 << 29


def listed():
    return [
        # One token's two experts at decode: 8 MB of weights, so launch and pipeline latency count.
        {"name": "grouped_token", "op": "grouped", "dtype": "bfloat16", "rows": 2, "experts": 8, "active": 2,
         "k": 2048, "n": 1024, "b_transposed": False, "skew": 0.0},
        # A decode batch over many experts: a few rows each, the weights' bytes are the time.
        {"name": "grouped_decode", "op": "grouped", "dtype": "bfloat16", "rows": 96, "experts": 32, "active": 30,
         "k": 2048, "n": 1408, "b_transposed": True, "skew": 0.5},
        # Half precision, many small ragged experts, widths that no tile divides, several experts without rows.
        {"name": "grouped_ragged", "op": "grouped", "dtype": "float16", "rows": 1511, "experts": 64, "active": 57,
         "k": 1544, "n": 2056, "b_transposed": False, "skew": 0.7},
        # A prefill chunk through the up projection.
        {"name": "grouped_prefill", "op": "grouped", "dtype": "bfloat16", "rows": 4109, "experts": 16, "active": 16,
         "k": 2048, "n": 4096, "b_transposed": True, "skew": 0.5},
        # A training step's rows: the tensor cores' rate is the time.
        {"name": "grouped_train", "op": "grouped", "dtype": "bfloat16", "rows": 32768, "experts": 8, "active": 8,
         "k": 4096, "n": 4096, "b_transposed": False, "skew": 0.3},
        # Weight gradient of a small layer.
        {"name": "wgrad_small", "op": "wgrad", "dtype": "bfloat16", "rows": 509, "experts": 8, "active": 7,
         "k": 1024, "n": 1024, "skew": 0.5},
        # Weight gradient of many small ragged experts in half precision: the written gradients' bytes count.
        {"name": "wgrad_ragged", "op": "wgrad", "dtype": "float16", "rows": 8111, "experts": 64, "active": 60,
         "k": 2048, "n": 1544, "skew": 0.7},
        # Weight gradient of the training step above.
        {"name": "wgrad_train", "op": "wgrad", "dtype": "bfloat16", "rows": 32768, "experts": 8, "active": 8,
         "k": 4096, "n": 4096, "skew": 0.3},
        # One token through a square projection: 8 MB of 4-bit weights.
        {"name": "w4_token", "op": "w4", "dtype": "bfloat16", "rows": 1, "experts": 1, "active": 1,
         "k": 4096, "n": 4096, "group": 128, "zeros": False, "skew": 0.0},
        # One token through a wide projection with zero points and short groups.
        {"name": "w4_wide", "op": "w4", "dtype": "float16", "rows": 1, "experts": 1, "active": 1,
         "k": 8192, "n": 16384, "group": 64, "zeros": True, "skew": 0.0},
        # A small decode batch, an odd number of outputs, the shortest groups.
        {"name": "w4_batch", "op": "w4", "dtype": "bfloat16", "rows": 15, "experts": 1, "active": 1,
         "k": 4096, "n": 11009, "group": 32, "zeros": False, "skew": 0.0},
        # A decode batch over 4-bit experts.
        {"name": "w4_experts", "op": "w4", "dtype": "bfloat16", "rows": 40, "experts": 32, "active": 22,
         "k": 4096, "n": 2048, "group": 128, "zeros": True, "skew": 0.4},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["grouped", "grouped", "wgrad", "w4", "w4"])
    while True:
        case = {"op": op, "dtype": rng.choice(["bfloat16", "float16"]), "skew": round(rng.uniform(0.0, 0.7), 2)}
        if op == "w4":
            case["experts"] = rng.choice([1, 1, rng.randint(2, 64)])
            case["rows"] = _log(rng, 1, 16) if case["experts"] == 1 else _log(rng, 1, 64)
            case["group"] = rng.choice([32, 64, 128])
            case["k"] = case["group"] * max(1, _log(rng, 512, 8192) // case["group"])
            case["n"] = _log(rng, 512, 16384)
            case["zeros"] = rng.random() < 0.5
        else:
            case["experts"] = _log(rng, 2, 64)
            case["rows"] = _log(rng, 1 if op == "grouped" else 64, 32768)
            case["k"] = 8 * _log(rng, 64, 1024)
            case["n"] = 8 * _log(rng, 64, 1024)
            if op == "grouped":
                case["b_transposed"] = rng.random() < 0.5
        case["active"] = min(case["rows"], rng.randint((case["experts"] + 1) // 2, case["experts"]))
        # The padded plain form and the 32-bit copies of the weights stay within the largest listed case's.
        if case["rows"] * case["k"] * case["n"] <= MAX_MACS // 2 and case["experts"] * case["k"] * case["n"] <= MAX_WEIGHTS:
            return case


def _dtype(case):
    return getattr(torch, case["dtype"])


def _counts(case, gen):
    """Rows of each expert: `active` of them hold one row or more, the others none."""
    experts, active, rows = case["experts"], case["active"], case["rows"]
    share = torch.exp(case["skew"] * torch.randn(active, generator=gen, dtype=torch.float64))
    picks = torch.multinomial(share, max(rows - active, 1), replacement=True, generator=gen)[: rows - active]
    counts = torch.zeros(experts, dtype=torch.int64)
    counts[torch.randperm(experts, generator=gen)[:active]] = 1 + torch.bincount(picks, minlength=active)
    return counts


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _dtype(case)
    experts, rows, k, n = case["experts"], case["rows"], case["k"], case["n"]
    counts = _counts(case, host)
    starts = torch.cumsum(counts, 0) - counts
    expert = torch.repeat_interleave(torch.arange(experts), counts)
    # The routing's plan: where each expert's rows begin, and each row's expert and place among its expert's rows.
    state = {
        "case": case,
        "cap": int(counts.max()),
        "offsets": torch.cat([starts, counts.sum().reshape(1)]).to(device=device, dtype=torch.int32),
        "expert": expert.to(device),
        "place": (torch.arange(rows) - starts[expert]).to(device),
    }

    def normal(*shape, scale=1.0):
        # In pieces of one leading index, so that the 32-bit draft of a large stack is never whole.
        out = torch.empty(shape, device=device, dtype=dtype)
        for piece in out if len(shape) == 3 else [out]:
            piece.copy_(torch.randn(piece.shape, device=device, generator=gen) * scale)
        return out

    if case["op"] == "grouped":
        state["a"] = normal(rows, k)
        state["b"] = normal(*((experts, n, k) if case["b_transposed"] else (experts, k, n)), scale=k ** -0.5)
        state["out"] = torch.empty(rows, n, device=device, dtype=dtype)
    elif case["op"] == "wgrad":
        state["a"] = normal(rows, k)
        state["grad"] = normal(rows, n)
        state["out"] = torch.empty(experts, k, n, device=device, dtype=dtype)
    else:
        groups = k // case["group"]
        state["a"] = normal(rows, k)
        state["q"] = torch.randint(0, 256, (experts, n, k // 2), device=device, dtype=torch.uint8, generator=gen)
        spread = 0.5 + torch.rand(experts, n, groups, device=device, generator=gen)
        state["scales"] = (spread * (k ** -0.5 / 4.6)).to(dtype)
        state["zeros"] = None
        if case["zeros"]:
            state["zeros"] = torch.randint(5, 11, (experts, n, groups), device=device, dtype=torch.uint8, generator=gen)
        state["out"] = torch.empty(rows, n, device=device, dtype=dtype)
    return state


def _padded(state, x):
    """Rows in 32 bits, laid out (experts, cap, width) with zeros after each expert's last row."""
    out = torch.zeros(state["case"]["experts"], state["cap"], x.shape[1], device=x.device, dtype=torch.float32)
    out[state["expert"], state["place"]] = x.float()
    return out


def _plain(state):
    case = state["case"]
    dtype = _dtype(case)
    if case["op"] == "wgrad":
        return torch.bmm(_padded(state, state["a"]).transpose(1, 2), _padded(state, state["grad"])).to(dtype)
    if case["op"] == "grouped":
        b = state["b"].float()
        b = b.transpose(1, 2) if case["b_transposed"] else b
    else:
        experts, n, k, group = case["experts"], case["n"], case["k"], case["group"]
        q = torch.stack([state["q"] & 15, state["q"] >> 4], -1).reshape(experts, n, k // group, group).float()
        zeros = 8.0 if state["zeros"] is None else state["zeros"].float().unsqueeze(-1)
        b = ((q - zeros) * state["scales"].float().unsqueeze(-1)).reshape(experts, n, k).transpose(1, 2)
    return torch.bmm(_padded(state, state["a"]), b)[state["expert"], state["place"]].to(dtype)


def _own(state):
    from teamredbench_b200 import kernels

    case = state["case"]
    if case["op"] == "grouped":
        return kernels.grouped_gemm(state["a"], state["b"], state["offsets"], state["out"],
                                    b_transposed=case["b_transposed"])
    if case["op"] == "wgrad":
        return kernels.grouped_gemm_wgrad(state["a"], state["grad"], state["offsets"], state["out"])
    if case["experts"] == 1:
        zeros = None if state["zeros"] is None else state["zeros"][0]
        return kernels.gemv_w4(state["a"], state["q"][0], state["scales"][0], state["out"], zeros=zeros)
    return kernels.gemv_w4(state["a"], state["q"], state["scales"], state["out"], zeros=state["zeros"],
                           offsets=state["offsets"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    rows, k, n, experts, active = case["rows"], case["k"], case["n"], case["experts"], case["active"]
    flops = 2.0 * rows * k * n
    offsets = 4 * (experts + 1) if experts > 1 else 0
    if case["op"] == "wgrad":  # the gradient of an expert without rows is written too, as zeros
        return {"bytes": 2 * (rows * (k + n) + experts * k * n) + offsets, "flops": flops}
    if case["op"] == "grouped":
        return {"bytes": 2 * (rows * (k + n) + active * k * n) + offsets, "flops": flops}
    weights = active * n * (k // 2 + (k // case["group"]) * (3 if case["zeros"] else 2))
    return {"bytes": weights + 2 * rows * (k + n) + offsets, "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    bounds = state["offsets"].tolist()
    x = state["a"].double()
    if case["op"] == "wgrad":
        out = torch.zeros(state["out"].shape, device=x.device, dtype=torch.float64)
    else:
        out = torch.empty(state["out"].shape, device=x.device, dtype=torch.float64)
    for e in range(case["experts"]):
        r = slice(bounds[e], bounds[e + 1])
        if bounds[e] == bounds[e + 1]:
            continue
        if case["op"] == "wgrad":
            out[e] = x[r].T @ state["grad"][r].double()
        elif case["op"] == "grouped":
            w = state["b"][e].double()
            out[r] = x[r] @ (w.T if case["b_transposed"] else w)
        else:
            packed = state["q"][e].long()
            w = torch.empty(case["n"], case["k"], device=x.device, dtype=torch.float64)
            w[:, 0::2] = (packed % 16).double()
            w[:, 1::2] = (packed // 16).double()
            z = 8 if state["zeros"] is None else state["zeros"][e].double().repeat_interleave(case["group"], 1)
            out[r] = x[r] @ ((w - z) * state["scales"][e].double().repeat_interleave(case["group"], 1)).T
    return out
