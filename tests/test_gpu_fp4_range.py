"""GPU tests of microscaled 4-bit floating point at the ends of the scales' range."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

from teamredbench_b200.kernels import dequantize_fp4, quantize_fp4  # noqa: E402
from tests.fp4_helpers import DTYPES, values  # noqa: E402


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
def test_every_value_is_exact_rounded_or_infinite(dtype):
    """All codes under all scales but NaN: one rounding in f16, none in bf16 and float32, infinite above each type."""
    scales = torch.zeros(255, 16, device="cuda", dtype=torch.uint8)
    scales[:, 0] = torch.arange(255)
    q = torch.arange(16, device="cuda", dtype=torch.uint8).mul(0x11).expand(255, 16).contiguous()
    out = dequantize_fp4(q, scales, torch.empty(255, 32, device="cuda", dtype=dtype)).double()
    want = values(q, scales)
    large = want.abs() >= (65520.0 if dtype is torch.float16 else 2.0 ** 128)  # f16 rounds from 65520 on up to 65536
    assert torch.equal(out, torch.where(large, torch.copysign(torch.tensor(float("inf"), device="cuda"), want).double(),
                                        want.to(dtype).double()))
    if dtype is not torch.float16:
        assert torch.equal(out[~large], want[~large])
        assert large[:253].sum() == 0 and large[253].any() and large[254].any()


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
def test_the_largest_values_come_back_finite(dtype):
    x = torch.full((3, 32), torch.finfo(dtype).max, device="cuda", dtype=dtype)
    x[1] = -x[1]
    x[2, 1:] = 0.0
    q, scales = torch.empty(3, 16, device="cuda", dtype=torch.uint8), torch.empty(3, 16, device="cuda", dtype=torch.uint8)
    quantize_fp4(x, q, scales)
    assert scales[:, 0].max() <= 252
    back = dequantize_fp4(q, scales, torch.empty(3, 32, device="cuda"))
    power = 2.0 ** (15 if dtype is torch.float16 else 127)  # max is just below twice this: 6 quarters of it
    assert torch.equal(back, x.float().sign() * 1.5 * power)
