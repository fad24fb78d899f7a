"""What the block-scaled E4M3 operators and the sorted rows refuse, told on the host: no GPU needed."""
import ctypes

import pytest
import torch

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    from gridbook_b200 import _native
    return _native.load()


def _text(lib):
    return lib.gb_last_error().decode()


P = ctypes.c_void_p(4096)          # an aligned address that no call below gets as far as reading
ODD = ctypes.c_void_p(4097)
NULL = ctypes.c_void_p(0)


@pytest.mark.parametrize("args,word", [
    ((P, P, P, P, P, 0, 4, 8, 24, 0, NULL), "multiple of 16"),
    ((P, P, P, P, P, 3, 4, 8, 128, 0, NULL), "dtype"),
    ((P, P, P, P, P, 0, -1, 8, 128, 0, NULL), "shape"),
    ((P, P, P, P, P, 0, 4, 0, 128, 0, NULL), "shape"),
    ((P, P, P, P, P, 0, 4, 8, 0, 0, NULL), "shape"),
    ((P, P, NULL, P, P, 0, 4, 8, 128, 0, NULL), "null"),
    ((ODD, P, P, P, P, 0, 4, 8, 128, 0, NULL), "aligned"),
    ((P, ODD, P, P, P, 0, 4, 8, 128, 0, NULL), "misaligned"),
    ((P, P, P, P, ODD, 0, 4, 8, 128, 0, NULL), "aligned"),
    ((P, P, P, P, P, 0, 1 << 31, 8, 128, 0, NULL), "too large"),
])
def test_gemm_refuses(lib, args, word):
    assert lib.gb_gemm_fp8_blocks(*args) != 0
    assert word in _text(lib)


@pytest.mark.parametrize("args,word", [
    ((P, P, P, P, P, 0, P, 0, 4, 8, 128, 0, NULL), "expert count"),
    ((P, P, P, P, P, 1025, P, 0, 4, 8, 128, 0, NULL), "expert count"),
    ((P, P, P, P, P, 1024, P, 0, 4, 1 << 22, 128, 0, NULL), "too large"),
    ((P, P, P, P, P, 4, P, 0, 4, 8, 120, 0, NULL), "multiple of 16"),
])
def test_grouped_gemm_refuses(lib, args, word):
    assert lib.gb_gemm_fp8_blocks_grouped(*args) != 0
    assert word in _text(lib)


def test_one_launch_linear_refuses(lib):
    def call(x=P, dtype=0, ld=128, rule=0, out=0, M=4, N=8, K=128):
        return lib.gb_linear_fp8_blocks(x, dtype, ld, rule, P, P, P, out, M, N, K, NULL)
    for kw, code, word in ((dict(M=5), 3, "4 rows"), (dict(x=ODD), 3, "4 rows"), (dict(ld=132), 3, "4 rows"), (dict(dtype=4), 1, "dtype"), (dict(rule=2), 1, "rule"),
                           (dict(ld=64), 1, "shorter"), (dict(K=24), 1, "multiple of 16"), (dict(out=9), 1, "dtype"), (dict(N=0), 1, "shape")):
        assert call(**kw) == code and word in _text(lib), kw


def test_empty_calls_launch_nothing(lib):
    before = lib.gb_launch_count()
    assert lib.gb_gemm_fp8_blocks(NULL, NULL, NULL, NULL, NULL, 0, 0, 8, 128, 0, NULL) == 0
    assert lib.gb_gemm_fp8_blocks_grouped(NULL, NULL, NULL, NULL, NULL, 4, NULL, 0, 0, 8, 128, 0, NULL) == 0
    assert lib.gb_fp8_quantize_blocks(NULL, 0, 128, 0, 128, 0, NULL, NULL, NULL) == 0
    assert lib.gb_moe_permute(NULL, 2, 64, NULL, NULL, 0, 2, 64, NULL, NULL) == 0
    assert lib.gb_moe_unpermute(NULL, 0, NULL, NULL, 0, 2, 64, NULL, NULL) == 0
    assert lib.gb_moe_unpermute_grad(NULL, NULL, 0, NULL, NULL, NULL, 0, 2, 64, NULL, NULL, NULL) == 0
    assert lib.gb_launch_count() == before


@pytest.mark.parametrize("args,word", [
    ((P, 5, 128, 4, 128, 0, P, P, NULL), "dtype"),
    ((P, 0, 128, 4, 128, 7, P, P, NULL), "scale rule"),
    ((P, 0, 64, 4, 128, 0, P, P, NULL), "shorter"),
    ((P, 0, 128, 4, 0, 0, P, P, NULL), "shape"),
    ((NULL, 0, 128, 4, 128, 0, P, P, NULL), "null"),
    ((ODD, 0, 128, 4, 128, 0, P, P, NULL), "misaligned"),
    ((P, 0, 1 << 20, 1 << 20, 1 << 20, 0, P, P, NULL), "too many blocks"),
])
def test_quantiser_refuses(lib, args, word):
    assert lib.gb_fp8_quantize_blocks(*args) != 0
    assert word in _text(lib)


def test_sorted_rows_refuse(lib):
    assert lib.gb_moe_permute(P, 1, 64, P, P, 4, 2, 64, P, NULL) != 0 and "bytes" in _text(lib)
    assert lib.gb_moe_permute(P, 2, 32, P, P, 4, 2, 64, P, NULL) != 0 and "shorter" in _text(lib)
    assert lib.gb_moe_permute(P, 2, 64, P, P, 4, 0, 64, P, NULL) != 0 and "shape" in _text(lib)
    assert lib.gb_moe_permute(P, 2, 64, P, P, 1 << 29, 4, 64, P, NULL) != 0 and "pairs" in _text(lib)
    assert lib.gb_moe_permute(P, 2, 64, P, NULL, 4, 2, 64, P, NULL) != 0 and "null" in _text(lib)
    assert lib.gb_moe_unpermute(P, 3, P, P, 4, 2, 64, P, NULL) != 0 and "dtype" in _text(lib)
    assert lib.gb_moe_unpermute(ODD, 0, P, P, 4, 2, 64, P, NULL) != 0 and "misaligned" in _text(lib)
    assert lib.gb_moe_unpermute_grad(P, NULL, 0, P, P, P, 4, 2, 64, NULL, P, NULL) != 0 and "null" in _text(lib)
    assert lib.gb_moe_swiglu_fp8(P, 0, 64, NULL, 4, 64, 0, P, P, NULL) != 0 and "shorter" in _text(lib)
    assert lib.gb_moe_permute_fp8(P, 0, 64, P, NULL, 4, 2, 64, 0, P, P, NULL) != 0 and "null" in _text(lib)


def test_one_launch_sort_refuses(lib):
    assert [lib.gb_moe_sort_applies(*a) for a in ((0, 4), (1, 0), (1, 1), (65536, 1024), (65537, 4), (8, 1025))] == [0, 0, 1, 1, 0, 0]
    assert lib.gb_moe_sort(P, 2, 8, 4, 0, P, P, P, P, NULL) != 0 and "bytes" in _text(lib)
    assert lib.gb_moe_sort(P, 4, 65537, 4, 0, P, P, P, P, NULL) == 3 and "gb_moe_route_inv" in _text(lib)
    assert lib.gb_moe_sort(P, 8, 8, 4, 0, P, P, P, NULL, NULL) != 0 and "null" in _text(lib)


def test_host_tensors_are_refused():
    from gridbook_b200 import kernels
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    q, s = torch.zeros(2, 128, dtype=E4M3), torch.zeros(2, 1)
    w, ws = torch.zeros(128, 128, dtype=E4M3), torch.zeros(1, 1)
    one = torch.zeros(2, dtype=torch.int32)
    srt = kernels.MoESort(one, one, one, one, 1)
    for call in (lambda: kernels.fp8_quantize_blocks(x), lambda: kernels.linear_fp8_blocks(x, w, ws), lambda: kernels.gemm_fp8_blocks(q, s, w, ws),
                 lambda: kernels.gemm_fp8_blocks_grouped(q, s, w[None], ws[None], one), lambda: kernels.moe_sort(one.view(2, 1), 4),
                 lambda: kernels.moe_permute(x, srt), lambda: kernels.moe_unpermute(x, srt), lambda: kernels.moe_permute_fp8(x, srt),
                 lambda: kernels.moe_swiglu_fp8(x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_rounding_of_the_plain_form_is_the_formats():
    """The tests' own E4M3 rounding against torch's on every representable value and every midpoint."""
    from tests.blocks import e4m3_round
    grid = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    grid = grid[torch.isfinite(grid)].sort().values
    mid = (grid[1:] + grid[:-1]) / 2
    v = torch.cat([grid, mid, mid + 1e-4, mid - 1e-4])
    assert torch.equal(e4m3_round(v), v.float().to(E4M3).double())


def test_layers_refuse_what_does_not_fit():
    from gridbook_b200.block_fp8 import BlockFP8Linear, BlockFP8MoE
    w, s = torch.zeros(200, 272, dtype=E4M3), torch.ones(2, 3)
    with pytest.raises(ValueError, match="multiple of 16"):
        BlockFP8Linear(200, 64)
    lin = BlockFP8Linear(272, 200)
    with pytest.raises(RuntimeError, match="before load"):
        lin(torch.zeros(1, 272))
    for a, b in ((w.float(), s), (w[:128], s), (w, s[:1]), (w, s.int())):
        with pytest.raises(ValueError):
            lin.load(a, b, "cpu")
    for args in ((4, 250, 128), (4, 256, 100), (0, 256, 128), (1025, 256, 128)):
        with pytest.raises(ValueError):
            BlockFP8MoE(*args)
    moe = BlockFP8MoE(2, 256, 128)
    w13, s13, w2, s2 = torch.zeros(2, 256, 256, dtype=E4M3), torch.ones(2, 2, 2), torch.zeros(2, 256, 128, dtype=E4M3), torch.ones(2, 2, 1)
    for args in ((w13[:1], s13, w2, s2), (w13, s13[:, :1], w2, s2), (w13, s13, w2.half(), s2), (w13, s13, w2, s2[..., :0])):
        with pytest.raises(ValueError):
            moe.load(*args, "cpu")


def test_operators_trace_without_running():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from gridbook_b200 import ops  # noqa: F401
    with FakeTensorMode():
        x = torch.empty(3, 5, 256, dtype=torch.bfloat16)
        y = torch.ops.prismaquant.fp8_blocks_linear(x, torch.empty(200, 256, dtype=E4M3), torch.empty(2, 2))
        assert y.shape == (3, 5, 200) and y.dtype is torch.bfloat16
        z = torch.ops.prismaquant.fp8_blocks_moe(x, torch.empty(2, 256, 256, dtype=E4M3), torch.empty(2, 2, 2), torch.empty(2, 256, 128, dtype=E4M3),
                                                 torch.empty(2, 2, 1), torch.empty(15, 2), torch.empty(15, 2, dtype=torch.int32), 0)
        assert z.shape == x.shape
