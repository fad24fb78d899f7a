"""The linear that quantises its rows inside the product, where a CTA walks several tiles and its rings come round many times: any number of
blocks, odd ones among them, against the same product of rows that were quantised first."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("N,K", [(80000, 1152), (151936, 896), (24000, 5760), (60000, 1408), (30000, 4224), (100001, 128), (70000, 16), (50000, 272),
                                 (45000, 1664), (20000, 2944), (60000, 1024)])
def test_tiles_one_after_the_other(dev, M, N, K):
    """Equal bit for bit, in fp32, time after time: the same sums in the same order, whatever order the slabs are multiplied in."""
    from gridbook_b200 import _native, kernels
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    w, sw = B.weights((N, K), g, dev)
    xs = [torch.randn(M, K, generator=g, device=dev).to(t) for t in (torch.bfloat16, torch.float16, torch.float32)]
    want = [kernels.gemm_fp8_blocks(*kernels.fp8_quantize_blocks(x), w, sw, out_dtype=torch.float32) for x in xs]
    ref = B.dequant_weight(w[-300:], sw[(N - 300) // 128:]) if (N - 300) % 128 == 0 else B.dequant_weight(w, sw)[-300:]
    B.assert_product(want[0][:, -300:], B.dequant_rows(*kernels.fp8_quantize_blocks(xs[0])), ref, f"{M}x{N}x{K}")
    del ref
    for i in range(24):
        assert torch.equal(kernels.linear_fp8_blocks(xs[i % 3], w, sw, out_dtype=torch.float32), want[i % 3]), f"call {i}"
    torch.cuda.synchronize()
    _native.prepare(0)
    assert _native.device_status(0) == 0
