"""A relu's result and its gradient's mask: what is above zero has a gradient, and nothing else."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("residual", [None, "rows", "apart"])
@pytest.mark.parametrize("M,N,K,dtype", [(256, 16384, 7232, HF), (256, 16384, 7232, BF), (251, 8195, 8192, HF), (40, 16384, 8192, BF), (2, 300, 1024, HF)])
def test_result_and_mask_agree_in_every_element(M, N, K, dtype, residual):
    """The bias' gradient adds up a column's mask; powers of two as the gradient of eight rows at a time tell them apart, exactly (255 is
    a bf16 number).  A residual of zeros leaves the sign to be seen."""
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    w = (torch.randn(N, K, generator=g, device=dev) / math.sqrt(K)).to(dtype)
    b = (0.1 * torch.randn(N, generator=g, device=dev)).to(dtype).requires_grad_()
    r = None if residual is None else torch.zeros(M, N + 3, dtype=dtype, device=dev)[:, 3 if residual == "apart" else 0:][:, :N]
    if residual == "rows":
        r = r.contiguous()
    y = kernels.linear_act(x, w, b, activation="relu", residual=r)
    powers = 2.0 ** (torch.arange(M, device=dev) % 8)
    wrong = 0
    for m in range(0, M, 8):
        dy = torch.zeros(M, N, dtype=dtype, device=dev)
        rows = slice(m, min(m + 8, M))
        dy[rows] = powers[rows, None].to(dtype)
        db, = torch.autograd.grad(y, b, dy, retain_graph=True)
        mask = (db.int()[None, :] >> torch.arange(rows.stop - m, device=dev)[:, None]) & 1
        wrong += int((mask.bool() != (y.detach()[rows] > 0)).sum())
    assert wrong == 0


def test_residuals_are_added_to_what_the_mask_says():
    """With a residual the result is that of the product without one plus the residual, each rounded once: no further apart than both
    roundings."""
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(5)
    M, N, K = 200, 4099, 7232
    x, w = torch.randn(M, K, generator=g, device=dev).to(HF).requires_grad_(), (torch.randn(N, K, generator=g, device=dev) / math.sqrt(K)).to(HF)
    r = torch.randn(M, N, generator=g, device=dev).to(HF)
    one, two = kernels.linear_act(x, w, activation="relu").double(), kernels.linear_act(x, w, activation="relu", residual=r).double()
    want = one + r.double()
    assert bool(((two - want).abs() <= 2.0 ** -11 * (one + want.abs()) * (1 + 2.0 ** -10) + 2.0 ** -24).all())
