"""Zeros keep their sign through the block quantisers: the bytes of E4M3(x / scale), not only its values."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _bytes(x, rule):
    """Bytes of the quotients, which B.quantize rounds as values: its zeros get the sign of x."""
    q, s = B.quantize(x, rule)
    return torch.where(q == 0, torch.where(torch.signbit(x.float().cpu()), 0x80, 0).to(torch.uint8), q.to(torch.float32).to(E4M3).view(torch.uint8)), s


def _rows(dtype, M, K, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=dev) * torch.exp2(torch.randint(-14, 15, (M, K), generator=g, device=dev).float())
    pick = torch.randint(0, 4, (M, K), generator=g, device=dev)
    x = torch.where(pick == 0, torch.zeros_like(x), torch.where(pick == 1, -torch.zeros_like(x), x))
    x[0] = -0.0                                                       # whole blocks of them
    x[-1, ::2] = 0.0
    x[-1, 1::2] = -0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(5, 256), (40, 5120), (33, 139)])
@pytest.mark.parametrize("rule", ["recip", "div"])
def test_signs_of_zeros(dev, dtype, M, K, rule):
    from gridbook_b200 import kernels
    x = _rows(dtype, M, K, dev, M + K)
    q, s = kernels.fp8_quantize_blocks(x, rule)
    rq, rs = _bytes(x, rule)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.view(torch.uint8).cpu(), rq)
    ids = torch.arange(M, device=dev, dtype=torch.int32).flip(0).view(M, 1)
    p, ps = kernels.moe_permute_fp8(x, kernels.moe_sort(ids, M), rule)
    assert torch.equal(p.view(torch.uint8).cpu(), rq.flip(0)) and torch.equal(ps.cpu(), rs.flip(0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_signs_of_zeros_between_the_projections(dev, dtype):
    """silu(gate) * up of a zero factor is a zero of the factors' signs."""
    from gridbook_b200 import kernels
    h = torch.tensor([[0.0, -0.0, 0.0, -0.0, 2.0, -2.0, 2.0, -2.0] * 32 + [1.0, 1.0, -1.0, -1.0, 0.0, 0.0, -0.0, -0.0] * 32], device=dev).to(dtype)
    h[0, 7], h[0, 256 + 7] = 3.0, 3.0                                 # a block with a value, and one of zeros alone
    q, _ = kernels.moe_swiglu_fp8(h)
    gate, up = h[0].double().chunk(2)
    v = gate / (1 + torch.exp(-gate)) * up
    zero = v == 0
    assert torch.equal(q[0].view(torch.uint8)[zero] == 0x80, torch.signbit(v)[zero]) and not bool((q[0].view(torch.uint8)[~zero] & 0x7F == 0).any())


@pytest.mark.parametrize("rule", ["recip", "div"])
def test_quotients_over_the_range_of_fp32(dev, rule):
    """Blocks whose largest magnitudes lie anywhere in fp32, with values down to its least beside them."""
    from gridbook_b200 import kernels
    g = torch.Generator(device=dev).manual_seed(5)
    M = 4000
    top = torch.exp2(torch.rand(M, 1, generator=g, device=dev) * 250 - 124)
    x = torch.randn(M, 128, generator=g, device=dev).clamp(-4, 4) / 4 * top
    x[:, 64:] *= torch.exp2(-torch.randint(0, 40, (M, 64), generator=g, device=dev).float())
    q, s = kernels.fp8_quantize_blocks(x, rule)
    rq, rs = _bytes(x, rule)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.view(torch.uint8).cpu(), rq)
