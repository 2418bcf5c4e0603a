"""GPU tests of the gradients of a weighted expert_dispatch: of x by expert_combine, of the weights by
expert_combine_grad, against the 64-bit formula and against differences."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200 import _native  # noqa: E402
from teamredbench_b200.kernels import expert_combine, expert_combine_grad, expert_dispatch, expert_sort  # noqa: E402

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
# Half of each type's smallest number.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


@pytest.fixture(autouse=True)
def no_device_error():
    assert _native.device_error(0, clear=True) == 0
    yield
    torch.cuda.synchronize()
    assert _native.device_error(0, clear=True) == 0


def _bound(dtype, ref, magnitude, terms):
    """One rounding to `dtype` of a sum of `terms` fp32 products: each product and each add drops at most 2^-24 of
    itself, and no partial sum is above `magnitude` by more than those errors."""
    err = 2 * (terms + 1) * 2.0 ** -24 * magnitude
    return err + torch.finfo(dtype).eps / 2 * (ref.abs() + err) + TINY[dtype]


# straight to registers; rows that begin anywhere; a CTA's and a warp's rings
@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("weights", ["own", "float32"])
@pytest.mark.parametrize("tokens, choices, width", [(1, 1, 8), (37, 3, 41), (300, 5, 2048), (4900, 2, 264)])
def test_gradients_of_a_weighted_dispatch(dtype, weights, tokens, choices, width):
    g = torch.Generator(device="cuda").manual_seed(width)

    def randn(*shape, dtype=torch.float64):
        return torch.randn(shape, device="cuda", dtype=torch.float64, generator=g).to(dtype)

    experts = 6
    ids = torch.randint(-1, experts, (tokens, choices), device="cuda", generator=g)
    _, slots = expert_sort(ids, torch.empty(experts + 1, device="cuda", dtype=torch.int32),
                           torch.empty(tokens, choices, device="cuda", dtype=torch.int32))
    here = slots >= 0
    rows = tokens * choices
    x, grad_out = randn(tokens, width, dtype=dtype), randn(rows, width, dtype=dtype)
    w = randn(tokens, choices, dtype=dtype if weights == "own" else torch.float32)
    grad_x, grad_w = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))

    at = torch.where(here.unsqueeze(-1), grad_out[slots.clamp_min(0).long()].double(), 0.0)  # of each choice
    factor = w.double().unsqueeze(-1)
    want_x, size_x = (factor * at).sum(1), (factor * at).abs().sum(1)
    products = x.double().unsqueeze(1) * at
    want_w, size_w = products.sum(-1), products.abs().sum(-1)

    out, again = torch.zeros_like(grad_out), grad_out.clone()
    expert_dispatch(x, slots, out, weights=w)
    expert_combine(grad_out, slots, grad_x, weights=w)
    expert_combine_grad(x, again, slots, w, again, grad_w)  # the gradient of out is not needed any more

    assert torch.equal(again[slots[here].long()], out[slots[here].long()])
    bound_x, bound_w = _bound(dtype, want_x, size_x, choices), _bound(w.dtype, want_w, size_w, width)
    assert ((grad_x.double() - want_x).abs() <= bound_x).all()
    assert ((grad_w.double() - want_w).abs() <= bound_w).all() and not grad_w[~here].any()

    # <gradient, direction> is the difference of two 64-bit dispatches along it, in each of which the result is linear; a
    # 64-bit sum of n terms is off by at most n * 2^-53 of the sum of their absolute values.
    def loss(x, w):
        return (torch.where(here.unsqueeze(-1), x.unsqueeze(1) * w.unsqueeze(-1), 0.0) * at).sum()

    dx, dw = randn(tokens, width), randn(tokens, choices)
    base, sums = loss(x.double(), w.double()), (size_w * (w.double().abs() + dw.abs())).sum() + (size_x * dx.abs()).sum()
    lost = 4 * tokens * choices * width * 2.0 ** -53 * sums
    assert ((grad_w.double() * dw).sum() - (loss(x.double(), w.double() + dw) - base)).abs() <= (bound_w * dw.abs()).sum() + lost
    assert ((grad_x.double() * dx).sum() - (loss(x.double() + dx, w.double()) - base)).abs() <= (bound_x * dx.abs()).sum() + lost
