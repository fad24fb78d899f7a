"""Block-scaled E4M3: the quantisers bit for bit, the GEMMs against fp64 products of the same operands, at the sizes where a tile, a
block, a slice of K or a segment ends, on other streams and in graphs."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _status():
    from gridbook_b200 import _native
    torch.cuda.synchronize()
    _native.prepare(0)
    assert _native.device_status(0) == 0


# ------------------------------------------------------------------ quantisers
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 5120), (3, 7), (5, 129), (17, 200), (4, 136), (2100, 1408), (300, 7168)])
@pytest.mark.parametrize("rule", ["recip", "div"])
def test_quantise_rows(dev, dtype, M, K, rule):
    from gridbook_b200 import kernels
    x = (torch.randn(M, K, generator=_gen(dev, M + K), device=dev) * torch.exp(2 * torch.randn(M, 1, generator=_gen(dev, K), device=dev))).to(dtype)
    q, s = kernels.fp8_quantize_blocks(x, rule)
    assert q.dtype is E4M3 and s.dtype is torch.float32
    rq, rs = B.quantize(x, rule)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(q.double().cpu(), rq)
    _status()


def test_quantise_edges(dev):
    """Blocks of zeros, of values under the floor, at the type's extremes, with an infinity or a NaN, signed zeros and ties."""
    from gridbook_b200 import kernels
    x = torch.zeros(9, 300, device=dev)
    x[1, :128] = 1e-12
    x[2] = torch.finfo(torch.float32).max
    x[3, 5] = float("inf")
    x[4, 290] = float("nan")
    x[5] = -0.0
    x[6, :17] = torch.arange(17, device=dev) * 0.0625 + 16.0        # ties between neighbours once 448 is there
    x[6, 17] = 448.0
    x[7, 128:256] = torch.randn(128, generator=_gen(dev, 1), device=dev) * 1e-38
    x[8, 0], x[8, 1] = torch.finfo(torch.float32).tiny, 3e38
    for rule in ("recip", "div"):
        q, s = kernels.fp8_quantize_blocks(x, rule)
        rq, rs = B.quantize(x, rule)
        assert torch.equal(s.cpu(), rs) or torch.equal(s.cpu().nan_to_num(-1), rs.nan_to_num(-1))
        assert torch.equal(torch.isnan(s.cpu()), torch.isnan(rs))
        v, r = q.double().cpu(), rq
        assert torch.equal(torch.isnan(v), torch.isnan(r))
        assert torch.equal(v.nan_to_num(0), r.nan_to_num(0))
    d = q.double().cpu() * s.cpu().double().repeat_interleave(128, 1)[:, :300]
    assert bool(torch.isnan(d[3, :128]).all()) and bool(torch.isfinite(d[3, 128:]).all())      # spreads over its block alone
    assert bool(torch.isnan(d[4, 256:]).all()) and bool(torch.isfinite(d[4, :256]).all())


def test_quantise_strided_rows_and_more_dimensions(dev):
    from gridbook_b200 import kernels
    base = torch.randn(40, 700, generator=_gen(dev, 2), device=dev).to(torch.bfloat16)
    for x in (base[:, 8:264], base[:, 3:131], base[::3, :256], base.t()[:256, :16], base[:1].expand(6, 700), base.view(2, 20, 700), base[0]):
        q, s = kernels.fp8_quantize_blocks(x)
        rq, rs = B.quantize(x)
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        assert torch.equal(s.cpu(), rs) and torch.equal(q.double().cpu(), rq)
    e = kernels.fp8_quantize_blocks(base[:0])
    assert e[0].shape == (0, 700) and e[1].shape == (0, 6)
    _status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("P,I,live", [(1, 768, 1), (7, 40, 5), (9, 131, 9), (700, 2048, 650), (3, 256, 0)])
def test_quantise_swiglu(dev, dtype, P, I, live):
    """scale: exp(-gate) is off by up to 2 + 1.173 |gate| units (CUDA's bound for the fast exponential) of 2^-23, the other
    six operations by a unit each.  A value: half an E4M3 step of its own (2^-4, or 2^-10 scales among the subnormals) on top."""
    from gridbook_b200 import kernels
    h = (torch.randn(P, 2 * I, generator=_gen(dev, P + I), device=dev) * 4).to(dtype)
    offsets = torch.tensor([0, live // 2, live], dtype=torch.int32, device=dev)
    q, s = kernels.moe_swiglu_fp8(h, offsets)
    g, u = h.double().chunk(2, -1)
    v = (g / (1 + torch.exp(-g)) * u)[:live]
    rel = (8 + 2 + 1.173 * float(g.abs().max())) * 2.0 ** -23
    amax = torch.nn.functional.pad(v, (0, -I % 128)).unflatten(-1, (-1, 128)).abs().amax(-1)
    rs = amax.clamp(min=1e-10) / 448
    assert bool(((s[:live].double() - rs).abs() <= rel * rs).all())
    step = B.spread(s[:live], I, -1)
    off = (q[:live].double() * step - v).abs()
    assert bool((off <= (2.0 ** -4 + rel) * v.abs() + 2.0 ** -10 * step * (1 + rel)).all())
    if live == P:                                                    # without offsets: every row
        q2, s2 = kernels.moe_swiglu_fp8(h)
        assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    _status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,topk,K,E,base", [(1, 8, 2048, 32, 0), (9, 2, 131, 4, 2), (700, 4, 256, 64, 0), (33, 1, 40, 3, 5)])
def test_quantise_into_expert_order(dev, dtype, T, topk, K, E, base):
    from gridbook_b200 import kernels
    g = _gen(dev, T * K)
    x = torch.randn(T, K, generator=g, device=dev).to(dtype)
    ids = torch.randint(-1, E + 2 * base, (T, topk), generator=g, device=dev, dtype=torch.int32)
    srt = kernels.moe_sort(ids, E, expert_base=base)
    q, s = kernels.moe_permute_fp8(x, srt)
    _, offsets, order, _ = B.sort(ids, E, base)
    rq, rs = B.quantize(x)
    n = offsets[-1]
    token = torch.tensor(order[:n], dtype=torch.long) // topk
    assert torch.equal(s[:n].cpu(), rs[token]) and torch.equal(q[:n].double().cpu(), rq[token])
    assert not bool(q[n:].view(torch.uint8).any()) and not bool(s[n:].any())
    _status()


# ------------------------------------------------------------------ dense product
SHAPES = [(1, 128, 128), (1, 1, 16), (1, 4096, 4096), (2, 200, 144), (5, 136, 640), (16, 512, 1536), (17, 130, 2064), (31, 384, 400), (33, 1000, 1040),
          (64, 256, 4096), (65, 77, 272), (100, 520, 1280), (128, 264, 5120), (129, 136, 256), (255, 256, 400), (256, 129, 128), (257, 384, 1168),
          (333, 1000, 2048), (700, 2056, 272), (2100, 4104, 384)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_product(dev, dtype, M, N, K):
    from gridbook_b200 import kernels
    g = _gen(dev, M + N + K)
    a, sa = B.rows(M, K, g, dev)
    w, sw = B.weights((N, K), g, dev)
    y = kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=dtype)
    assert y.dtype is dtype and y.shape == (M, N)
    _status()
    B.assert_product(y, B.dequant_rows(a, sa), B.dequant_weight(w, sw), f"{M}x{N}x{K}")


def test_product_scales_far_apart_and_special_values(dev):
    """Scales over many powers of two, a block of zeros, a NaN block that reaches its own row or features alone."""
    from gridbook_b200 import kernels
    for M in (3, 40, 300):
        g = _gen(dev, M)
        a, sa = B.rows(M, 640, g, dev)
        w, sw = B.weights((300, 640), g, dev)
        sa = sa * torch.exp2(torch.randint(-20, 20, sa.shape, generator=g, device=dev).float())
        sw = sw * torch.exp2(torch.randint(-20, 20, sw.shape, generator=g, device=dev).float())
        sa[1, 2] = 0.0
        y = kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=torch.float32)
        B.assert_product(y, B.dequant_rows(a, sa), B.dequant_weight(w, sw), f"rows {M}")
        sa[0, 4] = float("nan")
        sw[1, 0] = float("inf")
        y = kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=torch.float32)
        assert bool(torch.isnan(y[0]).all())
        fine = torch.isfinite(y[1:])
        assert bool(fine[:, :128].all()) and bool(fine[:, 256:].all()) and not bool(fine[:, 128:256].any())
    _status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (1, 136, 144), (4, 300, 400), (16, 1024, 1536), (40, 256, 4096), (200, 520, 640), (3, 520, 272),
                                   (13, 129, 2064), (7, 64, 16), (2, 256, 5120), (5, 40000, 256), (16, 33000, 400), (1, 30000, 4240), (9, 1, 7168)])
def test_linear(dev, dtype, M, N, K):
    from gridbook_b200 import kernels
    g = _gen(dev, M * N + K)
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    w, sw = B.weights((N, K), g, dev)
    q, s = B.quantize(x)
    y = kernels.linear_fp8_blocks(x, w, sw)
    assert y.dtype is dtype
    _status()
    B.assert_product(y, B.dequant_rows(q.to(dev), s.to(dev)), B.dequant_weight(w, sw), f"{M}x{N}x{K}")
    two = kernels.gemm_fp8_blocks(*kernels.fp8_quantize_blocks(x), w, sw, out_dtype=torch.bfloat16)
    assert torch.equal(two, kernels.linear_fp8_blocks(x, w, sw, out_dtype=torch.bfloat16))


def test_linear_views_dimensions_and_nothing(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 9)
    w, sw = B.weights((264, 512), g, dev)
    base = torch.randn(6, 600, generator=g, device=dev).to(torch.bfloat16)
    whole = kernels.linear_fp8_blocks(base[:, 40:552].contiguous(), w, sw)
    assert torch.equal(kernels.linear_fp8_blocks(base[:, 40:552], w, sw), whole)
    assert torch.equal(kernels.linear_fp8_blocks(base[:, 40:552].reshape(2, 3, 512), w, sw), whole.view(2, 3, 264))
    assert torch.equal(kernels.linear_fp8_blocks(base[2, 40:552], w, sw), kernels.linear_fp8_blocks(base[2:3, 40:552], w, sw)[0])
    assert kernels.linear_fp8_blocks(base[:0, :512], w, sw).shape == (0, 264)
    wt = w.view(torch.uint8).t().contiguous().t().view(E4M3)             # another order in memory
    assert torch.equal(kernels.linear_fp8_blocks(base[:, 40:552], wt, sw), whole)


def test_refusals(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 3)
    a, sa = B.rows(4, 256, g, dev)
    w, sw = B.weights((128, 256), g, dev)
    off = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    for call, kind in ((lambda: kernels.gemm_fp8_blocks(a.to(torch.bfloat16), sa, w, sw), TypeError), (lambda: kernels.gemm_fp8_blocks(a, sa.double(), w, sw), TypeError),
                       (lambda: kernels.gemm_fp8_blocks(a, sa[:, :1], w, sw), RuntimeError), (lambda: kernels.gemm_fp8_blocks(a, sa, w, sw[:, :1]), RuntimeError),
                       (lambda: kernels.gemm_fp8_blocks(a, sa, w[:, :128], sw[:, :1]), RuntimeError), (lambda: kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=torch.float64), TypeError),
                       (lambda: kernels.gemm_fp8_blocks(a[:, :24], sa[:, :1], w[:, :24], sw[:, :1]), RuntimeError),
                       (lambda: kernels.gemm_fp8_blocks(a, sa.cpu(), w, sw), RuntimeError),
                       (lambda: kernels.linear_fp8_blocks(torch.zeros(2, 128, device=dev), w, sw), RuntimeError),
                       (lambda: kernels.linear_fp8_blocks(torch.zeros(2, 256, device=dev, dtype=torch.float64), w, sw), TypeError),
                       (lambda: kernels.gemm_fp8_blocks_grouped(a, sa, w[None], sw[None], off.long()), RuntimeError),
                       (lambda: kernels.gemm_fp8_blocks_grouped(a, sa, w[None], sw[None], off[:1]), RuntimeError),
                       (lambda: kernels.gemm_fp8_blocks_grouped(a, sa, w[None], sw[None], off, out=torch.empty(4, 127, device=dev)), RuntimeError),
                       (lambda: kernels.fp8_quantize_blocks(a), TypeError), (lambda: kernels.moe_swiglu_fp8(torch.zeros(2, 3, device=dev)), RuntimeError),
                       (lambda: kernels.moe_swiglu_fp8(torch.zeros(2, 4, device=dev), off.float()), RuntimeError)):
        with pytest.raises(kind):
            call()
    _status()


# ------------------------------------------------------------------ grouped product
GROUPED = [  # rows of each expert, N, K, rows behind the last segment
    ([1], 128, 128, 0), ([0, 1, 0], 136, 256, 0), ([1] * 8, 256, 2048, 0), ([0, 0, 3, 0, 17, 1, 0, 16], 200, 144, 5), ([40, 0, 1, 90], 384, 640, 0),
    ([64] * 4, 129, 272, 3), ([200, 10, 0, 130], 264, 400, 7), ([257, 0, 256, 300, 1], 520, 512, 0), ([100] * 3, 77, 160, 1), ([0, 0, 0], 128, 128, 4),
    ([2, 700], 1024, 256, 0), ([500, 3, 129], 250, 1040, 9),
]


@pytest.mark.parametrize("counts,N,K,behind", GROUPED)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_grouped_product(dev, dtype, counts, N, K, behind):
    from gridbook_b200 import kernels
    P, E = sum(counts) + behind, len(counts)
    g = _gen(dev, P + N + K)
    a, sa = B.rows(P, K, g, dev)
    w, sw = B.weights((E, N, K), g, dev)
    offsets = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32, device=dev)
    out = torch.full((P, N), 77.0, dtype=dtype, device=dev)
    y = kernels.gemm_fp8_blocks_grouped(a, sa, w, sw, offsets, out=out)
    assert y.data_ptr() == out.data_ptr()
    _status()
    bounds = offsets.tolist()
    A = B.dequant_rows(a, sa)
    for e in range(E):
        if counts[e]:
            B.assert_product(y[bounds[e]:bounds[e + 1]], A[bounds[e]:bounds[e + 1]], B.dequant_weight(w[e], sw[e]), f"expert {e} of {counts}")
    assert bool((y[bounds[-1]:] == 77.0).all())                       # rows behind the last segment stay as they were
    if not behind:
        assert torch.equal(kernels.gemm_fp8_blocks_grouped(a, sa, w, sw, offsets, out_dtype=dtype), y)


def test_grouped_equals_dense_by_expert_at_many_experts(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 4)
    E, N, K = 1024, 128, 256
    counts = torch.randint(0, 4, (E,), generator=g, device=dev)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    P = int(offsets[-1])
    a, sa = B.rows(P, K, g, dev)
    w, sw = B.weights((E, N, K), g, dev)
    y = kernels.gemm_fp8_blocks_grouped(a, sa, w, sw, offsets)
    seg = torch.repeat_interleave(torch.arange(E, device=dev), counts)
    ref = torch.bmm(B.dequant_rows(a, sa).unsqueeze(1), B.dequant_weight(w, sw)[seg].transpose(1, 2)).squeeze(1)
    _status()
    assert bool(((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-3 * ref.abs().mean()).all())


# ------------------------------------------------------------------ streams, graphs, repeated calls
def test_another_stream_graph_and_repetition(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 11)
    for M in (1, 24, 150):
        w, sw = B.weights((520, 1040), g, dev)
        xs = [torch.randn(M, 1040, generator=g, device=dev).to(torch.bfloat16) for _ in range(3)]
        eager = [kernels.linear_fp8_blocks(x, w, sw) for x in xs]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = [kernels.linear_fp8_blocks(x, w, sw) for x in xs]
        side.synchronize()
        for p, q in zip(eager, other):
            assert torch.equal(p, q)
        x = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = kernels.linear_fp8_blocks(x, w, sw)
            z = kernels.linear_fp8_blocks(x, w, sw)
        for i in (1, 2, 0):
            x.copy_(xs[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager[i]) and torch.equal(z, eager[i])
    _status()


def test_weights_written_right_before_the_call(dev):
    """The product may fetch weights while the quantiser runs, not before what wrote them has finished."""
    from gridbook_b200 import kernels
    g = _gen(dev, 12)
    ws = [B.weights((4096, 4096), g, dev) for _ in range(2)]
    x = torch.randn(1, 4096, generator=g, device=dev).to(torch.bfloat16)
    want = [kernels.linear_fp8_blocks(x, *w) for w in ws]
    w, s = ws[0][0].clone(), ws[0][1].clone()
    for i in range(40):
        w.view(torch.uint8).copy_(ws[i % 2][0].view(torch.uint8))
        s.copy_(ws[i % 2][1])
        assert torch.equal(kernels.linear_fp8_blocks(x, w, s), want[i % 2])
        q, sq = kernels.fp8_quantize_blocks(x)
        assert torch.equal(kernels.gemm_fp8_blocks(q, sq, w, s), want[i % 2])
    _status()


# ------------------------------------------------------------------ offsets outside the rows, and past 32 bits
@pytest.mark.parametrize("P,E", [(200, 4), (1000, 2)])                  # few and many rows an expert: both kernels
def test_segments_are_taken_within_the_rows(dev, P, E):
    from gridbook_b200 import kernels
    g = _gen(dev, P)
    N, K = 264, 272
    a, sa = B.rows(P, K, g, dev)
    w, sw = B.weights((E, N, K), g, dev)
    inside = torch.tensor([0] * E + [P], dtype=torch.int32, device=dev)
    outside = torch.tensor([-5] + [0] * (E - 1) + [P + 1000], dtype=torch.int32, device=dev)
    want = kernels.gemm_fp8_blocks_grouped(a, sa, w, sw, inside)
    assert torch.equal(kernels.gemm_fp8_blocks_grouped(a, sa, w, sw, outside), want)
    B.assert_product(want, B.dequant_rows(a, sa), B.dequant_weight(w[-1], sw[-1]), "last expert")
    _status()


def test_rows_past_two_gigabytes(dev):
    """More than 2^31 values of x, of q and of the product; the last rows are looked at."""
    from gridbook_b200 import kernels
    g = _gen(dev, 21)
    M, K = 140000, 16384
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=dev)
    x[-3:] = torch.randn(3, K, generator=g, device=dev).to(torch.bfloat16)
    q, s = kernels.fp8_quantize_blocks(x)
    few, fs = kernels.fp8_quantize_blocks(x[-3:])
    assert torch.equal(q[-3:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(s[-3:], fs)
    assert not bool(q[-100:-3].view(torch.uint8).any())
    del q, s
    w, sw = B.weights((64, K), g, dev)
    y = kernels.linear_fp8_blocks(x, w, sw)
    B.assert_product(y[-3:], B.dequant_rows(few, fs), B.dequant_weight(w, sw), "last rows")
    assert not bool(y[-100:-3].any())
    del x, y
    a, sa = B.rows(70000, 16, g, dev)
    w, sw = B.weights((32768, 16), g, dev)
    y = kernels.gemm_fp8_blocks(a, sa, w, sw)
    assert y.numel() > 2 ** 31
    B.assert_product(y[-3:], B.dequant_rows(a[-3:], sa[-3:]), B.dequant_weight(w, sw), "last rows of a large product")
    _status()


def test_weights_past_four_gigabytes(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 22)
    E, N, K = 257, 4096, 4096
    w = torch.zeros(E, N, K, dtype=torch.float8_e4m3fn, device=dev)
    sw = torch.ones(E, N // 128, K // 128, device=dev)
    one, s1 = B.weights((N, K), g, dev)
    w[-1].view(torch.uint8).copy_(one.view(torch.uint8))
    sw[-1] = s1
    for P in (6, 257 * 80):
        a, sa = B.rows(P, K, g, dev)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=dev)
        offsets[-1] = P
        y = kernels.gemm_fp8_blocks_grouped(a, sa, w, sw, offsets)
        B.assert_product(y[-6:], B.dequant_rows(a[-6:], sa[-6:]), B.dequant_weight(one, s1), f"{P} rows")
    _status()


def test_more_slots_than_half_a_warp(dev):
    """A token's row written to twenty places."""
    from gridbook_b200 import kernels
    g = _gen(dev, 23)
    T, topk, K, E = 37, 20, 272, 64
    ids = torch.stack([torch.randperm(E, generator=g, device=dev)[:topk] for _ in range(T)]).to(torch.int32)
    ids[::3, 17] = -1
    x = torch.randn(T, K, generator=g, device=dev).to(torch.bfloat16)
    r = kernels.moe_sort(ids, E)
    q, s = kernels.moe_permute_fp8(x, r)
    fq, fs = kernels.fp8_quantize_blocks(x)
    live = int(r.offsets[-1])
    token = (r.order[:live] // topk).long()
    assert torch.equal(q[:live].view(torch.uint8), fq.view(torch.uint8)[token]) and torch.equal(s[:live], fs[token])
    assert not bool(q[live:].view(torch.uint8).any()) and not bool(s[live:].any())
    _status()


@pytest.mark.parametrize("M", [1, 2, 3, 4, 9, 16])
@pytest.mark.parametrize("N,K", [(128, 9008), (300, 17408), (5120, 17408), (20000, 1040)])
def test_linear_more_blocks_than_stages(dev, M, N, K):
    """Rings that are gone round several times, with one tile a CTA and with several."""
    from gridbook_b200 import kernels
    g = _gen(dev, M + N + K)
    w, sw = B.weights((N, K), g, dev)
    x = torch.randn(M, K, generator=g, device=dev).to(torch.bfloat16)
    q, s = kernels.fp8_quantize_blocks(x)
    want = kernels.gemm_fp8_blocks(q, s, w, sw, out_dtype=torch.float32)
    B.assert_product(want, B.dequant_rows(q, s), B.dequant_weight(w, sw), "product")
    y = kernels.linear_fp8_blocks(x, w, sw, out_dtype=torch.float32)
    B.assert_product(y, B.dequant_rows(q, s), B.dequant_weight(w, sw), "linear")
    for _ in range(20):
        assert torch.equal(kernels.linear_fp8_blocks(x, w, sw, out_dtype=torch.float32), y)
    _status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K", [(2500, 2048), (1300, 4990)])
def test_many_tokens_into_expert_order(dev, dtype, T, K):
    """Enough blocks that a half warp takes two, in rows of whole and of ragged blocks."""
    from gridbook_b200 import kernels
    g = _gen(dev, T)
    topk, E = 3, 24
    ids = torch.rand(T, E + 4, generator=g, device=dev).topk(topk, -1)[1]
    x = torch.randn(T, K, generator=g, device=dev).to(dtype)
    r = kernels.moe_sort(ids, E, expert_base=2)
    q, s = kernels.moe_permute_fp8(x, r)
    fq, fs = kernels.fp8_quantize_blocks(x)
    live = int(r.offsets[-1])
    token = (r.order[:live] // topk).long()
    assert 0 < live < T * topk
    assert torch.equal(q[:live].view(torch.uint8), fq.view(torch.uint8)[token]) and torch.equal(s[:live], fs[token])
    assert not bool(q[live:].view(torch.uint8).any()) and not bool(s[live:].any())
    _status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N", [(1300, 4099), (1300, 4098), (1300, 4100), (1300, 4104), (300, 1003), (300, 1004), (300, 1006), (300, 1016), (2500, 1030)])
def test_product_rows_of_every_alignment(dev, dtype, M, N):
    """Rows of D that are whole 16-byte pieces, words, single values: on pairs, single CTAs and slices of K; nothing beside them is written."""
    from gridbook_b200 import kernels
    g = _gen(dev, M + N)
    a, sa = B.rows(M, 1040, g, dev)
    w, sw = B.weights((N, 1040), g, dev)
    y = kernels.gemm_fp8_blocks(a, sa, w, sw, out_dtype=dtype)
    B.assert_product(y, B.dequant_rows(a, sa), B.dequant_weight(w, sw), f"{M}x{N}")
    counts = [M // 2 - 7, 0, M - M // 2 - 4]                            # eleven rows behind the last segment
    offsets = torch.tensor([0, counts[0], counts[0], sum(counts)], dtype=torch.int32, device=dev)
    out = torch.full((M, N), 77.0, dtype=dtype, device=dev)
    kernels.gemm_fp8_blocks_grouped(a, sa, w.unsqueeze(0).repeat(3, 1, 1), sw.unsqueeze(0).repeat(3, 1, 1), offsets, out=out)
    B.assert_product(out[:M - 11], B.dequant_rows(a[:M - 11], sa[:M - 11]), B.dequant_weight(w, sw), f"grouped {M}x{N}")
    assert bool((out[M - 11:] == 77.0).all())
    _status()
