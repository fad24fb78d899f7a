"""The renormalised sigmoid choice whose chosen scores are all small: weights and gradient are of ordinary size."""
import pytest
import torch

from tests.blocks import HALF

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("low", [-80.0, -88.0])
@pytest.mark.parametrize("E", [8, 300, 1500])
def test_small_scores_renormalised(dtype, low, E):
    """A score is off by four units of 2^-24 (exponential, sum, quotient) and by half a step of the subnormal fp32 numbers, another four
    at 2^-128; a chosen share by both, its own and the sum's, and a unit an addition and for the quotient; the gradient's difference by that of the
    shares relative to the largest weight's gradient."""
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(E)
    T, k, scale = 12, 4, 2.5
    l = torch.full((T, E), -120.0, dtype=dtype, device=dev)
    for t in range(T):
        l[t, torch.randperm(E, generator=g, device=dev)[:k]] = torch.tensor([low, low + 0.5, low + 1.0, low + 1.5], device=dev).to(dtype)
    dw = torch.randn(T, k, generator=g, device=dev) * (64.0 if dtype is torch.float16 else 65536.0)
    a = l.clone().requires_grad_()
    w, ids = kernels.moe_topk(a, k, score="sigmoid", renormalize=True, scale=scale)
    x = l.double().requires_grad_()
    c = torch.sigmoid(x).gather(1, ids.long())
    q = c / c.sum(-1, keepdim=True)
    want = scale * q
    assert torch.equal(ids.long(), torch.sort(l.double(), dim=-1, descending=True, stable=True).indices[:, :k])
    assert bool(((w.double() - want).abs() <= 32 * U * want).all())
    got, = torch.autograd.grad(w, a, dw)
    ref, = torch.autograd.grad(want, x, dw.double())
    size = torch.zeros_like(ref).scatter_(1, ids.long(), (scale * q * dw.double().abs().amax(-1, keepdim=True)).detach())
    assert bool(torch.isfinite(got).all())
    assert bool(((got.double() - ref).abs() <= 128 * U * size + HALF[dtype] * (1 + 128 * U) * ref.abs() + 2.0 ** -25).all())
