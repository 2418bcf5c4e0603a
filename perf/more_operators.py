"""Workloads around the products of an expert layer: rows to the experts and back, and 4-bit floating point.

Six kinds of pass, as a training or serving program of a mixture-of-experts model makes them:

``dispatch``  the router's choices sorted by expert, and every token's row copied to its experts' rows
``combine``   every token's output from its experts' rows, with the router's weights
``gradient``  of both: the gradients of the experts' rows, of the weights, and of the tokens' rows
``quantise``  rows to 4-bit floating point (e2m1) with one power-of-two scale (e8m0) a block of 32, and back
``product``   out[r] = B @ a[r] with both operands in 4-bit floating point
``experts``   tokens quantised straight into their experts' rows, then the product with each expert's 4-bit matrix

``slots[t, j]`` is the place of token t's choice j among the rows sorted by expert, -1 for a choice that no expert here takes.
"""
import math

import torch

own = False

MAX_MACS = 8192 ** 3
MAX_WEIGHTS = 1 << 28
MAX_MOVED = 16384 * 4 * 4096
MAX_QUANTISED = 16384 * 8192
BLOCK = 32
# What the codes of e2m1 stand for, without the sign, and the values half way between two of them.
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One token's two experts at decode: a few kilobytes, so launches and latency count.
        {"name": "dispatch_token", "op": "dispatch", "dtype": "bfloat16", "tokens": 1, "choices": 2, "experts": 8,
         "width": 2048, "absent": 0.0, "skew": 0.0},
        # A prefill chunk over many experts: each row is read once and written eight times.
        {"name": "dispatch_prefill", "op": "dispatch", "dtype": "bfloat16", "tokens": 4109, "choices": 8,
         "experts": 128, "width": 2048, "absent": 0.0, "skew": 0.5},
        # A decode batch back from its experts.
        {"name": "combine_decode", "op": "combine", "dtype": "bfloat16", "weights": "float32", "tokens": 40,
         "choices": 4, "experts": 32, "width": 4096, "absent": 0.0, "skew": 0.4},
        # A prefill chunk on one of two ranks that share the experts: half of the choices are the other rank's.
        {"name": "combine_prefill", "op": "combine", "dtype": "float16", "weights": "float16", "tokens": 8191,
         "choices": 4, "experts": 64, "width": 4096, "absent": 0.5, "skew": 0.5},
        # A small training step in 32 bits, rows of an odd length that no vector load divides.
        {"name": "gradient_small", "op": "gradient", "dtype": "float32", "weights": "float32", "tokens": 509,
         "choices": 8, "experts": 64, "width": 1001, "absent": 0.0, "skew": 0.7},
        # A training step's rows: two gigabytes moved.
        {"name": "gradient_train", "op": "gradient", "dtype": "bfloat16", "weights": "float32", "tokens": 16384,
         "choices": 4, "experts": 32, "width": 4096, "absent": 0.0, "skew": 0.3},
        # A decode batch's activations.
        {"name": "quantise_decode", "op": "quantise", "dtype": "bfloat16", "rows": 15, "k": 4096},
        # A weight matrix, when a model is loaded.
        {"name": "quantise_weights", "op": "quantise", "dtype": "bfloat16", "rows": 16384, "k": 8192},
        # A decode batch through a square projection: 8 MB of weights.
        {"name": "product_decode", "op": "product", "dtype": "bfloat16", "rows": 16, "n": 4096, "k": 4096},
        # The square product of the dense benchmark: the tensor cores' rate is the time.
        {"name": "product_square", "op": "product", "dtype": "bfloat16", "rows": 8192, "n": 8192, "k": 8192},
        # A decode batch over many experts, an odd number of outputs: a few rows each, the weights' bytes are the time.
        {"name": "experts_decode", "op": "experts", "dtype": "bfloat16", "tokens": 64, "choices": 4, "experts": 32,
         "n": 2047, "k": 4096, "absent": 0.0, "skew": 0.5},
        # A prefill chunk through the up projection.
        {"name": "experts_prefill", "op": "experts", "dtype": "float16", "tokens": 4109, "choices": 4, "experts": 16,
         "n": 4096, "k": 2048, "absent": 0.0, "skew": 0.5},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "gradient", "quantise", "product", "product", "experts", "experts"])
    while True:
        case = {"op": op, "dtype": rng.choice(["bfloat16", "float16"])}
        if op in ("product", "experts"):
            case["n"] = rng.choice([8 * _log(rng, 16, 1024), _log(rng, 128, 8192)])
            case["k"] = BLOCK * _log(rng, 4, 256)
        if op in ("dispatch", "combine", "gradient"):
            case["dtype"] = rng.choice(["bfloat16", "bfloat16", "float16", "float16", "float32"])
            case["width"] = rng.choice([8 * _log(rng, 16, 1024), 8 * _log(rng, 16, 1024), _log(rng, 128, 8192)])
        if op in ("combine", "gradient"):
            case["weights"] = rng.choice(["float32", case["dtype"]])
        if op in ("dispatch", "combine", "gradient", "experts"):
            case["tokens"] = _log(rng, 1, 16384)
            case["experts"] = _log(rng, 4, 256)
            case["choices"] = rng.randint(1, min(8, case["experts"]))
            case["absent"] = rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.9), 2)])
            case["skew"] = round(rng.uniform(0.0, 0.7), 2)
        elif op == "product":
            case["rows"] = _log(rng, 1, 8192)
        else:
            case["rows"] = _log(rng, 1, 16384)
            case["k"] = BLOCK * _log(rng, 1, 512)
        # A drawn case costs no more than the largest listed one of its kind, in the plain form's 32 bits too.
        if op == "product":
            if case["rows"] * case["n"] * case["k"] <= MAX_MACS and case["n"] * case["k"] <= MAX_WEIGHTS:
                return case
        elif op == "experts":
            rows = case["tokens"] * case["choices"]
            if (rows * case["n"] * case["k"] <= MAX_MACS // 2 and rows * max(case["n"], case["k"]) <= MAX_MOVED // 2
                    and case["experts"] * case["n"] * case["k"] <= MAX_WEIGHTS):
                return case
        elif op == "quantise":
            if case["rows"] * case["k"] <= MAX_QUANTISED:
                return case
        elif case["tokens"] * case["choices"] * case["width"] <= MAX_MOVED // (2 if case["dtype"] == "float32" else 1):
            return case


def _dtype(name):
    return getattr(torch, name)


def _pitch(k):
    """Bytes from one row's scales to the next one's: one byte a block, up to a multiple of 16."""
    return (k // BLOCK + 15) // 16 * 16


def _placed(case):
    """Choices that an expert here takes."""
    total = case["tokens"] * case["choices"]
    return total - int(total * case["absent"])


def _choices(case, device, gen):
    """Distinct experts a token, drawn by uneven shares; an exact number of the choices is another rank's (-1)."""
    tokens, choices, experts = case["tokens"], case["choices"], case["experts"]
    share = case["skew"] * torch.randn(experts, device=device, generator=gen)
    noise = torch.rand(tokens, experts, device=device, generator=gen).clamp_min(1e-20)
    ids = (share - torch.log(-torch.log(noise))).topk(choices, dim=1).indices  # int64, as a router's topk gives them
    gone = torch.randperm(tokens * choices, device=device, generator=gen)[_placed(case):]
    ids.view(-1)[gone] = -1
    return ids


def _sorted_by_expert(ids, experts):
    """(offsets, slots) by counting: a choice's place is its expert's start plus the earlier choices of that expert."""
    flat = ids.reshape(-1)
    one_hot = flat.unsqueeze(1) == torch.arange(experts, device=flat.device)
    running = torch.cumsum(one_hot, 0, dtype=torch.int32)
    ends = torch.cumsum(running[-1], 0, dtype=torch.int32)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    expert = flat.clamp_min(0)
    rank = running.gather(1, expert.unsqueeze(1)).squeeze(1) - 1
    slots = torch.where(flat >= 0, offsets[expert] + rank, -1)
    return offsets, slots.reshape(ids.shape).to(torch.int32)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _dtype(case["dtype"])
    state = {"case": case}

    def normal(*shape):
        # In pieces of at most 64 MB, so that the 32-bit draft of a large tensor is never whole.
        out = torch.empty(shape, device=device, dtype=dtype)
        for piece in out.split(max(1, (1 << 24) // shape[1])):
            piece.copy_(torch.randn(piece.shape, device=device, generator=gen))
        return out

    def blocks(*shape, centre):
        """Codes, all equally likely, and scales within a factor of two about 2^centre; past the last block, zeros."""
        k = shape[-1]
        q = torch.randint(0, 256, (*shape[:-1], k // 2), device=device, dtype=torch.uint8, generator=gen)
        scales = torch.zeros((*shape[:-1], _pitch(k)), device=device, dtype=torch.uint8)
        scales[..., :k // BLOCK] = torch.randint(126 + centre, 129 + centre, (*shape[:-1], k // BLOCK), device=device,
                                                 dtype=torch.uint8, generator=gen)
        return q, scales

    op = case["op"]
    if op in ("dispatch", "combine", "gradient", "experts"):
        tokens, choices = case["tokens"], case["choices"]
        rows = tokens * choices
        state["ids"] = _choices(case, device, gen)
        state["offsets"], state["slots"] = _sorted_by_expert(state["ids"], case["experts"])
        if op in ("combine", "gradient"):
            logits = torch.randn(tokens, choices, device=device, generator=gen)
            state["weights"] = torch.softmax(logits, 1).to(_dtype(case["weights"]))
    if op == "dispatch":
        state["x"] = normal(tokens, case["width"])
        state["out_offsets"], state["out_slots"] = state["offsets"].clone(), state["slots"].clone()
        state["rows"] = torch.zeros(rows, case["width"], device=device, dtype=dtype)
    elif op == "combine":
        state["y"] = normal(rows, case["width"])
        state["out"] = torch.empty(tokens, case["width"], device=device, dtype=dtype)
    elif op == "gradient":
        state["y"] = normal(rows, case["width"])
        state["grad"] = normal(tokens, case["width"])
        state["grad_y"] = torch.zeros_like(state["y"])
        state["grad_weights"] = torch.empty_like(state["weights"])
        # What came back through the experts' products, for the gradient of the tokens' rows.
        state["grad_rows"] = normal(rows, case["width"])
        state["grad_x"] = torch.empty_like(state["grad"])
    elif op == "quantise":
        # Activations and weights have rows and columns of very different sizes.
        state["x"] = normal(case["rows"], case["k"])
        state["x"] *= torch.exp(torch.randn(case["rows"], 1, device=device, generator=gen)).to(dtype)
        state["x"] *= torch.exp(0.5 * torch.randn(case["k"], device=device, generator=gen)).to(dtype)
        state["q"] = torch.empty(case["rows"], case["k"] // 2, device=device, dtype=torch.uint8)
        state["scales"] = torch.empty(case["rows"], _pitch(case["k"]), device=device, dtype=torch.uint8)
        state["out"] = torch.empty_like(state["x"])
    elif op == "product":
        state["a"], state["a_scales"] = blocks(case["rows"], case["k"], centre=-1)
        state["b"], state["b_scales"] = blocks(case["n"], case["k"], centre=-(3 + int(math.log2(case["k"])) // 2))
        state["out"] = torch.empty(case["rows"], case["n"], device=device, dtype=dtype)
    else:
        state["x"] = normal(tokens, case["k"])
        state["bounds"] = state["offsets"].tolist()
        state["a"] = torch.zeros(rows, case["k"] // 2, device=device, dtype=torch.uint8)
        state["a_scales"] = torch.zeros(rows, _pitch(case["k"]), device=device, dtype=torch.uint8)
        state["b"], state["b_scales"] = blocks(case["experts"], case["n"], case["k"],
                                               centre=-(2 + int(math.log2(case["k"])) // 2))
        state["out"] = torch.zeros(rows, case["n"], device=device, dtype=dtype)
    return state


def _place(rows, slots, values):
    """rows[slots[t, j]] = values[t] (or values[t, j]) where slots[t, j] is not -1."""
    here = slots >= 0
    if values.dim() == 2:
        values = values.unsqueeze(1).expand(-1, slots.shape[1], -1)
    rows[slots[here].long()] = values[here].to(rows.dtype)
    return rows


def _gathered(y, slots):
    """y's rows in 32 bits, (tokens, choices, width), zeros for a choice without a row."""
    rows = y[slots.clamp_min(0).long()].float()
    return torch.where((slots >= 0).unsqueeze(-1), rows, 0.0)


def _codes(x):
    """x (a float32 tensor) in blocks: (values on the levels of e2m1, powers of two), (..., k / 32, 32) and (..., k / 32, 1)."""
    x = x.unflatten(-1, (-1, BLOCK))
    largest = x.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(largest).exponent - 3).clamp(-127, 127)
    power = torch.exp2(exponent.double()).float()
    size = x.abs() * torch.exp2(-exponent.double()).float()  # exact
    level = torch.zeros_like(size)
    for i in range(1, len(LEVELS)):
        half_way = (LEVELS[i - 1] + LEVELS[i]) / 2
        # A tie goes to the level with the even code.
        reached = size >= half_way if i % 2 == 0 else size > half_way
        level = torch.where(reached, LEVELS[i], level)
    return torch.copysign(level, x), power


def _quantised(x):
    level, power = _codes(x.float())
    return (level * power).flatten(-2)


def _values(q, scales):
    """What codes and scales stand for, in 32 bits."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=q.device)
    values = torch.stack([levels[(q & 15).long()], levels[(q >> 4).long()]], -1).flatten(-2)
    blocks = values.shape[-1] // BLOCK
    power = torch.exp2(scales[..., :blocks].double() - 127).float()
    return (values.unflatten(-1, (blocks, BLOCK)) * power.unsqueeze(-1)).flatten(-2)


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "dispatch":
        offsets, slots = _sorted_by_expert(state["ids"], case["experts"])
        return offsets, slots, _place(state["rows"], slots, state["x"])
    if op == "combine":
        weights = state["weights"].float().unsqueeze(-1)
        return (weights * _gathered(state["y"], state["slots"])).sum(1).to(state["out"].dtype)
    if op == "gradient":
        slots, grad = state["slots"], state["grad"].float().unsqueeze(1)
        grad_y = _place(state["grad_y"], slots, state["weights"].float().unsqueeze(-1) * grad)
        grad_weights = (grad * _gathered(state["y"], slots)).sum(-1).to(state["weights"].dtype)
        grad_x = _gathered(state["grad_rows"], slots).sum(1).to(state["grad"].dtype)
        return grad_y, grad_weights, grad_x
    if op == "quantise":
        return torch.cat([_quantised(x).to(x.dtype) for x in state["x"].split(4096)])
    if op == "product":
        a, b = _values(state["a"], state["a_scales"]), _values(state["b"], state["b_scales"])
        return (a @ b.T).to(state["out"].dtype)
    x = _quantised(state["x"])
    rows = torch.zeros(state["a"].shape[0], case["k"], device=x.device)
    _place(rows, state["slots"], x)
    for e, (lo, hi) in enumerate(zip(state["bounds"][:-1], state["bounds"][1:])):
        if hi > lo:
            state["out"][lo:hi] = rows[lo:hi] @ _values(state["b"][e], state["b_scales"][e]).T
    return state["out"]


def _own(state):
    from teamredbench_b200 import kernels

    op = state["case"]["op"]
    if op == "dispatch":
        offsets, slots = kernels.expert_sort(state["ids"], state["out_offsets"], state["out_slots"])
        return offsets, slots, kernels.expert_dispatch(state["x"], slots, state["rows"])
    if op == "combine":
        return kernels.expert_combine(state["y"], state["slots"], state["out"], weights=state["weights"])
    if op == "gradient":
        kernels.expert_combine_grad(state["grad"], state["y"], state["slots"], state["weights"], state["grad_y"],
                                    state["grad_weights"])
        kernels.expert_combine(state["grad_rows"], state["slots"], state["grad_x"])
        return state["grad_y"], state["grad_weights"], state["grad_x"]
    if op == "quantise":
        kernels.quantize_fp4(state["x"], state["q"], state["scales"])
        return kernels.dequantize_fp4(state["q"], state["scales"], state["out"])
    if op == "product":
        return kernels.gemm_fp4(state["a"], state["a_scales"], state["b"], state["b_scales"], state["out"])
    kernels.quantize_fp4(state["x"], state["a"], state["a_scales"], slots=state["slots"])
    return kernels.gemm_fp4(state["a"], state["a_scales"], state["b"], state["b_scales"], state["out"],
                            offsets=state["offsets"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "float32" else 2
    if op in ("quantise", "product"):
        rows = case["rows"]
        if op == "quantise":  # x in, codes and scales out, their values out
            return {"bytes": rows * case["k"] * (2 * size + 0.5 + 1 / BLOCK), "flops": 4.0 * rows * case["k"]}
        blocks = (rows + case["n"]) * case["k"] * (0.5 + 1 / BLOCK)
        return {"bytes": blocks + 2 * rows * case["n"], "flops": 2.0 * rows * case["n"] * case["k"]}
    tokens, placed = case["tokens"], _placed(case)
    plan = 4 * tokens * case["choices"]
    if op == "experts":
        active = min(case["experts"], placed)
        rows = placed * case["k"] * (0.5 + 1 / BLOCK)
        weights = active * case["n"] * case["k"] * (0.5 + 1 / BLOCK)
        moved = 2 * tokens * case["k"] + plan + 2 * rows + weights + 4 * (case["experts"] + 1) + 2 * placed * case["n"]
        return {"bytes": moved, "flops": 2.0 * placed * case["n"] * case["k"] + 4.0 * tokens * case["k"]}
    row = size * case["width"]
    if op == "dispatch":
        return {"bytes": 3 * plan + 4 * (case["experts"] + 1) + (tokens + placed) * row, "flops": 0.0}
    weights = tokens * case["choices"] * (4 if case["weights"] == "float32" else 2)
    if op == "combine":
        return {"bytes": plan + weights + (tokens + placed) * row, "flops": 2.0 * placed * case["width"]}
    return {"bytes": 2 * plan + 2 * weights + (2 * tokens + 3 * placed) * row, "flops": 4.0 * placed * case["width"]}


def _exact_blocks(x):
    """The nearest values of the blocks' own grids, in 64 bits: a grid's step is 2^e at 2 to 4, and half or twice beside it."""
    x = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    largest = x.abs().max(-1, keepdim=True).values
    exponent = torch.frexp(largest.clamp_min(2.0 ** -125)).exponent.long() - 3
    unit = ((exponent + 1023) << 52).view(torch.float64)  # 2^exponent
    size = (x / unit).abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    near = torch.clamp(torch.round(size / step) * step, max=6.0)  # torch.round takes ties to the even multiple
    return (torch.sign(x) * near * unit).flatten(-2)


def _exact_values(q, scales):
    codes = torch.empty(*q.shape[:-1], 2 * q.shape[-1], device=q.device, dtype=torch.int64)
    codes[..., 0::2] = (q % 16).long()
    codes[..., 1::2] = (q // 16).long()
    exponent, mantissa = (codes // 2) % 4, codes % 2
    size = torch.where(exponent == 0, 0.5 * mantissa, torch.exp2((exponent - 1).double()) * (1 + 0.5 * mantissa))
    values = torch.where(codes >= 8, -size, size)
    blocks = values.shape[-1] // BLOCK
    return values * torch.exp2(scales[..., :blocks].double() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        return torch.cat([_exact_blocks(x) for x in state["x"].split(2048)])
    if op == "product":
        a, b = _exact_values(state["a"], state["a_scales"]), _exact_values(state["b"], state["b_scales"])
        return a @ b.T
    flat = state["ids"].reshape(-1)
    # Places by a stable sort; the choices of other ranks go behind the last expert.
    order = torch.sort(torch.where(flat < 0, case["experts"], flat), stable=True).indices[:_placed(case)]
    token = order // case["choices"]
    if op == "dispatch":
        slots = torch.full_like(flat, -1)
        slots[order] = torch.arange(order.numel(), device=flat.device)
        offsets = torch.searchsorted(flat[order], torch.arange(case["experts"] + 1, device=flat.device))
        rows = torch.zeros(state["rows"].shape, device=flat.device, dtype=torch.float64)
        rows[: order.numel()] = state["x"][token].double()
        return offsets.to(torch.int32), slots.reshape(state["ids"].shape).to(torch.int32), rows
    if op == "experts":
        out = torch.zeros(state["out"].shape, device=flat.device, dtype=torch.float64)
        x = _exact_blocks(state["x"])[token]
        expert = flat[order]
        for e in range(case["experts"]):
            mine = (expert == e).nonzero().squeeze(1)
            if mine.numel():
                out[mine] = x[mine] @ _exact_values(state["b"][e], state["b_scales"][e]).T
        return out
    weights = state["weights"].reshape(-1)[order].double()

    def added(y, factor=None):
        out = torch.zeros(case["tokens"], case["width"], device=flat.device, dtype=torch.float64)
        for j in range(case["choices"]):
            mine = (order % case["choices"] == j).nonzero().squeeze(1)  # at most one row a token
            part = y[mine].double()
            out[token[mine]] += part if factor is None else factor[mine].unsqueeze(1) * part
        return out

    if op == "combine":
        return added(state["y"], weights)
    grad_y = torch.zeros(state["y"].shape, device=flat.device, dtype=torch.float64)
    grad_weights = torch.zeros(flat.shape, device=flat.device, dtype=torch.float64)
    for piece in torch.arange(order.numel(), device=flat.device).split(8192):
        grad = state["grad"][token[piece]].double()
        grad_y[piece] = weights[piece].unsqueeze(1) * grad
        grad_weights[order[piece]] = (grad * state["y"][piece].double()).sum(1)
    return grad_y, grad_weights.reshape(state["ids"].shape), added(state["grad_rows"])
