"""The grouped block-scaled product with offsets that fall and rise again, which no sort makes: segments overlap, so that there are more tiles of
rows than rising offsets can have.  Nothing outside of the output is touched, no wait runs out, and with the same weights for every expert the
rows of the first segment are what they are."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from gridbook_b200 import _native
    _native.prepare(0)
    return torch.device("cuda:0")


@pytest.mark.parametrize("P,E,N,K", [(64, 64, 264, 4096), (8, 8, 128, 8192), (200, 4, 136, 4096), (1024, 32, 2056, 400), (3000, 12, 520, 640), (2000, 1024, 128, 256)])
def test_overlapping_segments(dev, P, E, N, K):
    from gridbook_b200 import _native, kernels
    lib = _native.load()
    g = torch.Generator(device=dev).manual_seed(P + E)
    a, sa = B.rows(P, K, g, dev)
    w1, s1 = B.weights((N, K), g, dev)
    w, s = w1.unsqueeze(0).repeat(E, 1, 1), s1.unsqueeze(0).repeat(E, 1, 1)
    offsets = torch.tensor([P * (e % 2) for e in range(E + 1)], dtype=torch.int32, device=dev)       # 0, P, 0, P, ...
    out = torch.full((P * N + 128,), 77.0, dtype=torch.bfloat16, device=dev)
    d = out[64:64 + P * N]
    for _ in range(3):
        _native.check(lib.gb_gemm_fp8_blocks_grouped(a.data_ptr(), sa.data_ptr(), w.data_ptr(), s.data_ptr(), offsets.data_ptr(), E, d.data_ptr(), 0, P, N, K, 0,
                                                     _native.stream_ptr(dev)), lib)
    torch.cuda.synchronize()
    assert _native.device_status(0) == 0
    B.assert_product(d.view(P, N), B.dequant_rows(a, sa), B.dequant_weight(w1, s1), f"{P} rows of {E} experts")
    assert bool((out[:64] == 77.0).all()) and bool((out[64 + P * N:] == 77.0).all())
    rising = torch.tensor([0] * E + [P], dtype=torch.int32, device=dev)                              # the last expert has all
    assert torch.equal(kernels.gemm_fp8_blocks_grouped(a, sa, w, s, rising), d.view(P, N))
