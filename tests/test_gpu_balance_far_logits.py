"""The balance loss of rows whose logits are far from zero: masks of the type's lowest value, padding, its largest; loss and gradient
against the 64-bit formula, beside ordinary rows."""
import pytest
import torch

from tests.blocks import HALF

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
FAR = {HF: (3e4, -3e4), BF: (1e10, -1e10, 1e18, -1e18), FP: (1e10, -1e10, 1e18, -1e18)}                      # their squares fit fp32
EXTREME = {HF: (65504.0, -65504.0), BF: (-1e30, 2.5e38, torch.finfo(BF).min, torch.finfo(BF).max), FP: (-1e30, 2.5e38, torch.finfo(FP).min, torch.finfo(FP).max)}


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _rows(values, E, dtype, dev):
    """Ordinary rows; for every value a row of it, one with half of it ordinary, one with an expert masked; ids at random."""
    g = torch.Generator(device=dev).manual_seed(E)
    l = (2.0 * torch.randn(40 + 3 * len(values), E, generator=g, device=dev)).to(dtype)
    for i, v in enumerate(values):
        l[3 * i] = v
        l[3 * i + 1, ::2] = v
        l[3 * i + 2] = v
        l[3 * i + 2, E // 2] = -float("inf")
    return l, torch.randint(0, E, (l.shape[0], 2), generator=g, device=dev)


def _check(l, ids, z_coef, coef=0.5, d_loss=3.0):
    """Errors, relative: the difference to the largest logit rounds by half a unit of itself, and so does its product, each times that
    difference in the exponential (terms past 100 are zeros in fp32, 64-bit ones below 1e-43), which is off by two units; sums of positive terms by a unit for each
    of up to 64 in a row, sums over the tokens by one for each of a group's."""
    from gridbook_b200 import kernels
    T, E = l.shape
    a = l.clone().requires_grad_()
    loss, counts = kernels.moe_balance_loss(a, ids, coef=coef, z_coef=z_coef)
    f = torch.bincount(ids.reshape(-1), minlength=E).double() / ids.numel()
    p, z = torch.softmax(l.double(), -1), torch.logsumexp(l.double(), -1, keepdim=True)
    want = coef * E * (f * p.mean(0)).sum() + z_coef * z.square().mean()
    value = float(loss.detach())
    assert torch.equal(counts.double(), torch.round(f * ids.numel()))
    tol = (2 * 100 + 64 + T + 16) * U
    if float(want) > torch.finfo(FP).max:
        assert value == float("inf")
    else:
        assert abs(value - float(want)) <= 2 * tol * float(want), (value, float(want))
    got, = torch.autograd.grad(loss, a, torch.tensor(d_loss, device=l.device))
    # by the formula: torch's derivative of logsumexp is exp(x - result), and past 1e16 the result holds no log E any more
    ref = d_loss / T * p * (coef * E * (f - (f * p).sum(-1, keepdim=True)) + 2.0 * z_coef * z)
    size = d_loss / T * p * (coef * E * (f + (f * p).sum(-1, keepdim=True)) + 2.0 * z_coef * z.abs())
    # results and exponentials below fp32's normal numbers count as nothing; fp16's own steps end at 2^-24
    bound = 8 * tol * size + (1 + 8 * tol) * HALF[l.dtype] * ref.abs() + (2.0 ** -25 if l.dtype is HF else 1e-35)
    off = (got.double() - ref).abs() - bound
    assert got.dtype is l.dtype and bool(torch.isfinite(got).all()) and float(off.max()) <= 0.0, float(off.max())


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("E", [6, 200, 300, 1000, 1500])
def test_rows_far_from_zero(dev, dtype, E):
    l, ids = _rows(FAR[dtype], E, dtype, dev)
    for z_coef in (0.0, 0.25):
        _check(l, ids, z_coef)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("E", [6, 200, 300, 1000, 1500])
def test_rows_at_the_ends_of_the_type(dev, dtype, E):
    """Where the squares of the z-loss pass fp32 the loss does, and the gradient, which has the first power, does not."""
    _check(*_rows(EXTREME[dtype], E, dtype, dev), 0.25)
