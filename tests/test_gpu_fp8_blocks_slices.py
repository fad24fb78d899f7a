"""The block-scaled product on single CTAs whose tiles split K over a cluster: sums that meet in one CTA's shared memory, an even and an
odd number of them, the last one short, rows of D of every alignment."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu

# Whole and ragged tiles of rows and features; two to five slices (how many clusters of five run at once differs from card to card)
SHAPES = [(333, 5120, 17408), (333, 2310, 8192), (300, 2311, 7184), (333, 3500, 3088), (600, 1284, 5136), (600, 1280, 5136), (640, 1273, 5632), (257, 2304, 5120),
          (129, 4872, 4096), (700, 1030, 16384)]


@pytest.fixture(scope="module")
def dev():
    from gridbook_b200 import _native
    _native.prepare(0)
    return torch.device("cuda:0")


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_product(dev, dtype, M, N, K):
    from gridbook_b200 import _native, kernels
    kernel, slices = kernels.gemm_fp8_blocks_kernel(M, N, K)
    assert kernel == "gemm_blocks_tile_kernel<1>" and slices > 1
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    a, sa = B.rows(M, K, g, dev)
    w, sw = B.weights((N, K), g, dev)
    y = kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=dtype)
    B.assert_product(y, B.dequant_rows(a, sa), B.dequant_weight(w, sw), f"{M}x{N}x{K}")
    for _ in range(10):                                              # sums in the order of K: the same bits each time
        assert torch.equal(kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=dtype), y)
    torch.cuda.synchronize()
    assert _native.device_status(0) == 0


def test_nothing_beside_the_product_is_written(dev):
    """The library's entry on an output between two guards."""
    from gridbook_b200 import _native, kernels
    lib = _native.load()
    g = torch.Generator(device=dev).manual_seed(7)
    for M, N, K in ((333, 2310, 8192), (300, 2311, 7184), (257, 2304, 5120)):
        a, sa = B.rows(M, K, g, dev)
        w, sw = B.weights((N, K), g, dev)
        for dtype, code in ((torch.bfloat16, 0), (torch.float32, 2)):
            out = torch.full((M * N + 128,), 77.0, dtype=dtype, device=dev)
            d = out[64:64 + M * N]
            _native.check(lib.gb_gemm_fp8_blocks(a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), d.data_ptr(), code, M, N, K, 0,
                                                 _native.stream_ptr(dev)), lib)
            assert torch.equal(d.view(M, N), kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=dtype))
            assert bool((out[:64] == 77.0).all()) and bool((out[64 + M * N:] == 77.0).all())


def test_streams_and_a_graph(dev):
    from gridbook_b200 import kernels
    g = torch.Generator(device=dev).manual_seed(8)
    pairs = [(*B.rows(333, 8192, g, dev), *B.weights((2310, 8192), g, dev)) for _ in range(2)]
    want = [kernels.gemm_fp8_blocks(*p) for p in pairs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.gemm_fp8_blocks(*pairs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    graph = torch.cuda.CUDAGraph()
    a, sa = pairs[0][0].clone(), pairs[0][1].clone()
    with torch.cuda.graph(graph):
        y = kernels.gemm_fp8_blocks(a, sa, *pairs[0][2:])
    for i in (1, 0):
        a.view(torch.uint8).copy_(pairs[i][0].view(torch.uint8))
        sa.copy_(pairs[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, kernels.gemm_fp8_blocks(*pairs[i][:2], *pairs[0][2:]))
