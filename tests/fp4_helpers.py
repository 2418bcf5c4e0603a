"""Plain forms of microscaled 4-bit floating point, written from the format's definition, and error bounds."""
from __future__ import annotations

import torch

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of the codes 0 to 7; 8 to 15 are their negatives


def pitch(k):
    return -(-(k // 32) // 16) * 16


def values(q, scales, device="cuda"):
    """What codes and scales stand for, in 64 bits."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=q.device)
    v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], -1).flatten(-2)
    code = scales[..., :v.shape[-1] // 32].double()
    power = torch.where(code == 255, float("nan"), torch.exp2(code - 127))
    return v * power.repeat_interleave(32, -1)


def quantised(x):
    """(codes one a value, scale bytes) of x, in 64 bits: the nearest of the 15 values, the even code at a tie."""
    x = x.double().unflatten(-1, (-1, 32))
    largest = x.abs().amax(-1)
    bad = ~x.isfinite().all(-1)
    exponent = torch.frexp(torch.where(bad | (largest == 0), 1.0, largest)).exponent - 3
    exponent = torch.where(largest == 0, -127, exponent.clamp_min(-127))
    size = torch.where(bad.unsqueeze(-1), 0.0, x.abs() * torch.exp2(-exponent.double()).unsqueeze(-1)).clamp_max(6.0)
    levels = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    distance = (size.unsqueeze(-1) - levels).abs()
    nearest = distance == distance.amin(-1, keepdim=True)
    even = torch.tensor([1, 0] * 4, dtype=torch.int32, device=x.device)
    code = (nearest.int() * (1 + even)).argmax(-1)  # of two nearest ones, the even
    negative = torch.where(bad.unsqueeze(-1), False, x.signbit())
    return (code + 8 * negative).flatten(-2), torch.where(bad, 255, exponent + 127)


def packed(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)


def operand(shape, seed, low=120, high=131, behind=None):
    """Random codes, scales 2^(low - 127) to 2^(high - 128), and `behind` (or any bytes) behind each row's last block."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = shape[-1]
    q = torch.randint(0, 256, (*shape[:-1], k // 2), device="cuda", dtype=torch.uint8, generator=g)
    scales = torch.randint(0, 256, (*shape[:-1], pitch(k)), device="cuda", dtype=torch.uint8, generator=g)
    if behind is not None:
        scales.fill_(behind)
    scales[..., :k // 32] = torch.randint(low, high, (*shape[:-1], k // 32), device="cuda", dtype=torch.uint8, generator=g)
    return q, scales


def product(a, b, bounds):
    """(result, sum of absolute products) of out[r] = b[e] @ a[r], NaN outside every group; a, b in 64 bits."""
    ref = torch.full((a.shape[0], b.shape[1]), float("nan"), dtype=torch.float64, device=a.device)
    magnitude = ref.clone()
    for e, (lo, hi) in enumerate(bounds):
        ref[lo:hi] = a[lo:hi] @ b[e].T
        magnitude[lo:hi] = a[lo:hi].abs() @ b[e].T.abs()
    return ref, magnitude


def check(got, ref, magnitude, terms):
    """One rounding to 16 bits, and a sum of `terms` products (exact in fp32: 4 x 4 bits and powers of two) whose fp32 adds
    may each drop the last bit (2^-23) of a partial sum, which `magnitude` bounds."""
    err = (terms + 16) * 2.0 ** -23 * magnitude
    half, tiny = torch.finfo(got.dtype).eps / 2, 2.0 ** -25 if got.dtype is torch.float16 else 0.0
    excess = (got.double() - ref).abs() - (err + half * (ref.abs() + err) + tiny)
    assert not got.isnan().any(), got.isnan().nonzero()[:3].tolist()
    worst = excess.max().item() if excess.numel() else 0.0
    assert worst <= 0.0, f"beyond the bound by {worst}, at {(excess == excess.max()).nonzero()[:3].tolist()}"
