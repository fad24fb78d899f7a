"""gelu's tail left of zero: as near as the erf's approximation, 1.5e-7 of one, and fp32's exponential let it be."""
import pytest
import torch

from tests.blocks import HALF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 300])
def test_tail(dtype, M):
    """Half of z times the tail of 1 + erf: that approximation's bound of 1.5e-7 times |z| / 2; the exponential's argument z^2 / 2 rounds by
    half a unit and its function by two units and 1.2 times that argument's size, the polynomial and products by some ten: of the value, up to
    100 units of 2^-24 at z = -12; half a step of the type, fp16's subnormal ones half of 2^-24."""
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    z = torch.linspace(-12, 0, 4000, device=dev).to(dtype)
    w = torch.zeros(z.numel(), 8, dtype=dtype, device=dev)
    w[:, 0] = z
    x = torch.zeros(M, 8, dtype=dtype, device=dev)
    x[:, 0] = 1.0
    y = kernels.linear_act(x, w, activation="gelu").double()
    zd = z.double()
    ref = 0.5 * zd * torch.special.erfc(-zd * 0.5 ** 0.5)
    err = 0.75e-7 * zd.abs() + 2.0 * 100 * 2.0 ** -24 * ref.abs()
    tol = err * (1 + 2.0 ** -8) + HALF[dtype] * (1 + 2.0 ** -8) * ref.abs() + (2.0 ** -25 if dtype is torch.float16 else 1e-38)
    assert bool(((y - ref).abs() <= tol).all())
