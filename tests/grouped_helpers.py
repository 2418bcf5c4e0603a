"""Plain 64-bit forms and error bounds for the grouped-product tests."""
from __future__ import annotations

import torch

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
# Half the spacing of 16-bit results around 1 (8 and 11 significant bits), and of float16's smallest numbers.
ROUNDOFF = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
SMALLEST = {"bfloat16": 0.0, "float16": 2.0 ** -25}


def offsets_of(counts, first=0, device="cuda"):
    total, out = first, [first]
    for c in counts:
        total += c
        out.append(total)
    return torch.tensor(out, dtype=torch.int32, device=device)


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])


def allowed(dtype, ref, magnitude, terms):
    """|result - ref| allowed: one rounding to 16 bits, and a sum of `terms` products whose fp32 adds may each drop
    the last bit (2^-23) of a partial sum, which `magnitude` (the sum of the products' absolute values) bounds."""
    err = (terms + 16) * 2.0 ** -23 * magnitude
    return err + ROUNDOFF[dtype] * (ref.abs() + err) + SMALLEST[dtype]


def check(dtype, got, ref, magnitude, terms):
    excess = (got.double() - ref).abs() - allowed(dtype, ref, magnitude, terms)
    worst = excess.max().item() if excess.numel() else 0.0
    assert worst <= 0.0, f"beyond the bound by {worst}, at {(excess == excess.max()).nonzero()[:3].tolist()}"


def bounds(offsets):
    o = offsets.tolist()
    return list(zip(o[:-1], o[1:]))


def product(a, b, offsets, b_transposed):
    """(result, sum of absolute products) of out[r] = a[r] @ b[e], NaN outside every group."""
    n = b.shape[1] if b_transposed else b.shape[2]
    ref = torch.full((a.shape[0], n), float("nan"), dtype=torch.float64, device=a.device)
    mag = ref.clone()
    for e, (lo, hi) in enumerate(bounds(offsets)):
        w = b[e].double().T if b_transposed else b[e].double()
        ref[lo:hi] = a[lo:hi].double() @ w
        mag[lo:hi] = a[lo:hi].double().abs() @ w.abs()
    return ref, mag


def wgrad(a, grad, offsets):
    ref = torch.zeros((offsets.numel() - 1, a.shape[1], grad.shape[1]), dtype=torch.float64, device=a.device)
    mag = ref.clone()
    for e, (lo, hi) in enumerate(bounds(offsets)):
        ref[e] = a[lo:hi].double().T @ grad[lo:hi].double()
        mag[e] = a[lo:hi].double().abs().T @ grad[lo:hi].double().abs()
    return ref, mag


def w4_operands(groups, n, k, group, dtype, seed, with_zeros):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (groups, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = randn((groups, n, k // group), dtype, seed + 1, 0.05)
    zeros = None
    if with_zeros:
        zeros = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8)
    return q, scales, zeros


def w4_weights(q, scales, zeros):
    """The weights that q, scales and zeros stand for, in 64 bits."""
    w = torch.stack([q & 15, q >> 4], -1).flatten(-2).double()
    group = w.shape[-1] // scales.shape[-1]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, -1)
    return (w - z) * scales.double().repeat_interleave(group, -1)
