"""Forward-mode derivatives of the sorted rows: there are none, and nobody gets a result that has lost them."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_tangents_are_refused():
    from gridbook_b200 import kernels
    one = torch.zeros(2, dtype=torch.int32)
    srt = kernels.MoESort(one, one, one, one, 1)
    x, w = torch.zeros(2, 128), torch.ones(2, 1)
    with fwd.dual_level():
        dx, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, torch.ones_like(w))
        for call in (lambda: kernels.moe_permute(dx, srt), lambda: kernels.moe_unpermute(dx, srt), lambda: kernels.moe_unpermute(dx, srt, w),
                     lambda: kernels.moe_unpermute(x, srt, dw)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_tangents_of_gradients_are_refused():
    """A gradient with a tangent (forward over reverse) would lose it in the backward pass."""
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(1)
    ids = torch.rand(6, 4, generator=g, device=dev).topk(2, -1)[1]
    srt = kernels.moe_sort(ids, 4)
    x = torch.randn(6, 64, generator=g, device=dev).requires_grad_()
    w = torch.rand(6, 2, generator=g, device=dev).requires_grad_()
    rows = kernels.moe_permute(x, srt)
    plain, weighted = kernels.moe_unpermute(rows, srt), kernels.moe_unpermute(rows, srt, w)
    with fwd.dual_level():
        for out, leaves in ((rows, [x]), (plain, [x]), (weighted, [x, w])):
            seed = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaves, seed, retain_graph=True)
    dx, dw = torch.autograd.grad(weighted, [x, w], torch.ones_like(weighted))          # and without one they are there
    assert torch.allclose(dx, w.sum(1, keepdim=True).expand_as(dx)) and torch.allclose(dw, x.sum(1, keepdim=True).expand_as(dw), atol=1e-4)
