"""Weights, scales and routes that were written right in front of the call, by copies and by a launch of this package that lets the next ones
start before it is done: the products fetch them while a quantiser still runs, which must not be before their writer has finished."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _through_permute(kernels, t, identity):
    """A copy of the rows of a matrix by the row permutation, which starts its dependents at once."""
    if t.dtype is E4M3:
        return kernels.moe_permute(t.view(torch.bfloat16), identity).view(E4M3)
    return kernels.moe_permute(t, identity)


@pytest.mark.parametrize("M", [1, 5, 16, 64, 100, 300, 700])
def test_linear(dev, M):
    from gridbook_b200 import kernels
    g = torch.Generator(device=dev).manual_seed(M)
    N, K = 4096, 4096
    ws = [B.weights((N, K), g, dev) for _ in range(2)]
    x = torch.randn(M, K, generator=g, device=dev).to(torch.bfloat16)
    want = [kernels.linear_fp8_blocks(x, *w) for w in ws]
    assert not torch.equal(*want)
    rows, blocks = (kernels.moe_sort(torch.arange(n, device=dev, dtype=torch.int32).view(n, 1) // 4, -(-n // 4)) for n in (N, N // 128))
    w, s = ws[0][0].clone(), ws[0][1].clone()
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        if i % 2:
            w.view(torch.uint8).copy_(ws[i // 2 % 2][0].view(torch.uint8))
            s.copy_(ws[i // 2 % 2][1])
            got.append((kernels.linear_fp8_blocks(x, w, s), i // 2 % 2))
        else:
            fresh = _through_permute(kernels, ws[i // 2 % 2][0], rows)
            scale = _through_permute(kernels, ws[i // 2 % 2][1], blocks)
            got.append((kernels.linear_fp8_blocks(x, fresh, scale), i // 2 % 2))
            fresh.view(torch.uint8).fill_(0x7F)                      # NaN wherever a later call finds its memory unwritten
            scale.fill_(float("nan"))
            del fresh, scale
    for y, i in got:
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("T", [1, 16, 300])
def test_routed_layer(dev, T):
    from gridbook_b200 import kernels
    g = torch.Generator(device=dev).manual_seed(T)
    E, H, I, topk = 16, 1024, 512, 4
    sets = [(*B.weights((E, 2 * I, H), g, dev), *B.weights((E, H, I), g, dev)) for _ in range(2)]
    routes = [torch.softmax(torch.randn(T, E, generator=g, device=dev), -1).topk(topk, -1) for _ in range(2)]
    x = torch.randn(T, H, generator=g, device=dev).to(torch.bfloat16)
    want = {(i, j): kernels.moe_fp8_blocks(x, *sets[i], *routes[j]) for i in range(2) for j in range(2)}
    held, ids, weights = [t.clone() for t in sets[0]], routes[0][1].clone(), routes[0][0].clone()
    torch.cuda.synchronize()
    got = []
    for n in range(32):
        i, j = n % 2, n // 2 % 2
        weights.copy_(routes[j][0])
        for to, t in zip(held, sets[i]):
            to.view(torch.uint8).copy_(t.view(torch.uint8))
        ids.copy_(routes[j][1])
        got.append((kernels.moe_fp8_blocks(x, *held, weights, ids), (i, j)))
    for y, key in got:
        assert torch.equal(y, want[key])
