"""Tokens sorted by expert and back, with their gradients: the sort and the copies exactly, sums against fp64, gradients against
their formulas and against differences of the forward pass."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CASES = [(1, 1, 8, 1, 0), (1, 8, 2048, 128, 0), (5, 3, 33, 7, 2), (64, 2, 1, 4, 0), (40, 6, 200, 16, 8), (300, 8, 768, 128, 0), (2000, 4, 130, 300, 0),
         (7, 12, 64, 5, 0)]           # tokens, top-k, width, experts held here, first of them


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _ids(T, topk, E, base, g, dev):
    return torch.randint(-1 if base else 0, E + 2 * base, (T, topk), generator=g, device=dev, dtype=torch.int32)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


@pytest.mark.parametrize("T,topk,H,E,base", CASES + [(3000, 2, 8, 20, 5), (1100, 4, 8, 256, 3), (1, 1, 8, 4096, 0), (1500, 3, 8, 700, 9), (513, 1, 8, 9, 0), (4100, 2, 8, 1024, 1),
                                                  (8192, 8, 8, 128, 0), (5000, 4, 8, 256, 100), (9000, 8, 8, 64, 3), (6000, 1, 8, 1500, 0)])
def test_sort(dev, T, topk, H, E, base):
    from gridbook_b200 import kernels
    ids = _ids(T, topk, E, base, _gen(dev, T + topk), dev)
    for i in (ids, ids.long(), ids.t().contiguous().t()):
        r = kernels.moe_sort(i, E, expert_base=base)
        counts, offsets, order, place = B.sort(ids, E, base)
        assert r.counts.tolist() == counts and r.offsets.tolist() == offsets and r.order.tolist() == order and r.place.tolist() == place
        assert r.topk == topk and r.place.dtype is torch.int32


def test_ids_of_other_types_and_past_32_bits(dev):
    from gridbook_b200 import kernels
    for T in (3, 40000):
        ids = torch.randint(0, 6, (T, 2), generator=_gen(dev, T), device=dev)
        want = kernels.moe_sort(ids.int(), 4, expert_base=1)
        far = torch.where(ids == 0, ids + (1 << 32) + 2, ids)        # held nowhere, whatever the low half says
        for i in (ids, far, ids.to(torch.int16), ids.to(torch.uint8)):
            got = kernels.moe_sort(i, 4, expert_base=1)
            for a, b in ((got.counts, want.counts), (got.offsets, want.offsets), (got.order, want.order), (got.place, want.place)):
                assert torch.equal(a, b)


def test_nothing_to_sort(dev):
    from gridbook_b200 import kernels
    r = kernels.moe_sort(torch.empty(0, 4, dtype=torch.int32, device=dev), 6)
    assert r.counts.tolist() == [0] * 6 and r.offsets.tolist() == [0] * 7 and r.order.numel() == 0
    x = torch.empty(0, 16, device=dev, requires_grad=True)
    rows = kernels.moe_permute(x, r)
    out = kernels.moe_unpermute(rows, r, torch.empty(0, 4, device=dev))
    assert rows.shape == (0, 16) and out.shape == (0, 16)
    out.sum().backward()
    assert x.grad.shape == (0, 16)
    # every pair held elsewhere: zeros, and zero gradients
    r = kernels.moe_sort(torch.full((3, 2), 9, dtype=torch.int32, device=dev), 4)
    x, w = torch.randn(3, 16, device=dev, requires_grad=True), torch.randn(3, 2, device=dev, requires_grad=True)
    rows = kernels.moe_permute(x, r)
    assert not bool(rows.any())
    out = kernels.moe_unpermute(rows, r, w)
    assert not bool(out.any())
    out.sum().backward()
    assert not bool(x.grad.any()) and not bool(w.grad.any())


def _plain(x, y, w, place, T, topk):
    """rows, out in fp64; rows that no pair has are zero."""
    P = T * topk
    live = place >= 0
    pair = torch.arange(P, device=place.device)[live]
    rows = torch.zeros(P, x.shape[1], dtype=torch.float64, device=x.device).index_put((place[live],), x.double()[pair // topk])
    out = torch.zeros(T, x.shape[1], dtype=torch.float64, device=x.device).index_put((pair // topk,), y.double()[place[live]] * w.double().reshape(-1)[pair, None],
                                                                                      accumulate=True)
    return rows, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,topk,H,E,base", CASES)
def test_rows_there_and_back_with_gradients(dev, dtype, T, topk, H, E, base):
    """A sum of n fp32 products: n units of 2^-24 of the sum of magnitudes (the products are fused), and half a step of the
    result's type."""
    from gridbook_b200 import kernels
    g = _gen(dev, T * H + topk)
    r = kernels.moe_sort(_ids(T, topk, E, base, g, dev), E, expert_base=base)
    n, place = int(r.offsets[-1]), r.place.long()
    x = torch.randn(T, H, generator=g, device=dev).to(dtype).requires_grad_()
    y = torch.randn(T * topk, H, generator=g, device=dev).to(dtype)
    y[n:] = float("nan")                                             # rows that no pair has count nothing
    y.requires_grad_()
    w = torch.rand(T, topk, generator=g, device=dev).requires_grad_()
    rows, out = kernels.moe_permute(x, r), kernels.moe_unpermute(y, r, w)
    assert rows.dtype is dtype and out.dtype is dtype
    x64, y64, w64 = (t.detach().double().requires_grad_() for t in (x, y, w))
    rows64, out64 = _plain(x64, y64, w64, place, T, topk)
    _, size = _plain(x, y.detach().abs(), w.detach(), place, T, topk)
    half = B.HALF[dtype]
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    assert torch.equal(rows.double(), rows64)
    assert bool(((out.double() - out64).abs() <= half * out64.abs() + 2 * topk * 2.0 ** -24 * size + tiny).all())
    d_rows = torch.randn(T * topk, H, generator=g, device=dev).to(dtype)
    d_out = torch.randn(T, H, generator=g, device=dev).to(dtype)
    got = torch.autograd.grad([rows, out], [x, y, w], [d_rows, d_out])
    want = torch.autograd.grad([rows64, out64], [x64, y64, w64], [d_rows.double(), d_out.double()])
    _, dx_size = _plain(x, d_rows.abs(), torch.ones_like(w), place, T, topk)
    assert bool(((got[0].double() - want[0]).abs() <= half * want[0].abs() + 2 * topk * 2.0 ** -24 * dx_size + tiny).all())
    assert bool(((got[1].double() - want[1]).abs() <= (half + 2.0 ** -23) * want[1].abs() + tiny).all())
    live = (place >= 0).view(T, topk)
    mag = (y.detach().double().abs()[place.clamp(min=0)].view(T, topk, H) * d_out.double().abs().unsqueeze(1)).sum(-1)
    assert bool(((got[2].double() - want[2]).abs() <= (H + 8) * 2.0 ** -24 * mag)[live].all())
    assert not bool(got[2][~live].any()) and not bool(got[1][n:].any())
    # ones as weights: the gradient is the permutation
    y2 = y.detach().clone().requires_grad_()
    ones = kernels.moe_unpermute(y2, r)
    _, ones64 = _plain(x, y, torch.ones_like(w), place, T, topk)
    assert bool(((ones.double() - ones64).abs() <= half * ones64.abs() + 2 * topk * 2.0 ** -24 * _plain(x, y.detach().abs(), torch.ones_like(w), place, T, topk)[1] + tiny).all())
    (d_y2,) = torch.autograd.grad(ones, y2, d_out)
    assert torch.equal(d_y2, kernels.moe_permute(d_out, r))


def test_gradients_against_differences(dev):
    """out is linear in y and in the weights: a central difference of any width is exact but for the rounding of the outputs, (top-k + 1)
    units of 2^-24 of the magnitudes each."""
    from gridbook_b200 import kernels
    g = _gen(dev, 77)
    T, topk, H, E = 20, 4, 96, 10
    r = kernels.moe_sort(_ids(T, topk, E, 2, g, dev), E, expert_base=2)
    x = torch.randn(T, H, generator=g, device=dev, requires_grad=True)
    w = torch.rand(T, topk, generator=g, device=dev, requires_grad=True)
    d_out = torch.randn(T, H, generator=g, device=dev)
    vx, vw = torch.randn(T, H, generator=g, device=dev), torch.randn(T, topk, generator=g, device=dev)
    f = lambda a, b: (kernels.moe_unpermute(kernels.moe_permute(a, r), r, b).double() * d_out.double()).sum()  # noqa: E731
    dx, dw = torch.autograd.grad(kernels.moe_unpermute(kernels.moe_permute(x, r), r, w), [x, w], d_out)
    with torch.no_grad():
        size = float((kernels.moe_unpermute(kernels.moe_permute(x.abs() + vx.abs(), r), r, w.abs() + vw.abs()).double() * d_out.double().abs()).sum())
        tol = 4 * (H + topk) * 2.0 ** -24 * size                     # the gradients' own sums on top
        assert abs(float((f(x + vx, w) - f(x - vx, w)) / 2 - (dx.double() * vx.double()).sum())) <= tol
        assert abs(float((f(x, w + vw) - f(x, w - vw)) / 2 - (dw.double() * vw.double()).sum())) <= tol


def test_strides_broadcasts_types_and_needs(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 5)
    T, topk, H, E = 12, 2, 80, 6
    r = kernels.moe_sort(_ids(T, topk, E, 0, g, dev), E)
    base = torch.randn(T, 300, generator=g, device=dev).to(torch.bfloat16)
    for x in (base[:, 8:88], base[:, 3:83], base.t()[:T, :12], base[:1, :H].expand(T, H), base[:, :H].view(3, 4, H)):
        assert torch.equal(kernels.moe_permute(x, r), kernels.moe_permute(x.contiguous().view(-1, x.shape[-1]), r))
    # a gradient that is a broadcast number, and only one of the inputs asking for one
    y, w = torch.randn(T * topk, H, generator=g, device=dev), torch.rand(T, topk, generator=g, device=dev)
    for need_y, need_w in ((True, False), (False, True), (True, True)):
        a, b = y.clone().requires_grad_(need_y), w.clone().requires_grad_(need_w)
        kernels.moe_unpermute(a, r, b).sum().backward()
        assert (a.grad is not None) == need_y and (b.grad is not None) == need_w
        if need_y:
            assert torch.equal(a.grad, w.reshape(-1)[r.order.long()][:, None].expand(-1, H))
        if need_w:
            want = y.double().sum(-1)[r.place.long()].view(T, topk)
            assert bool(((b.grad.double() - want).abs() <= (H + 8) * 2.0 ** -24 * y.double().abs().sum(-1)[r.place.long()].view(T, topk)).all())
    # weights of another type get their gradient in it
    h = w.to(torch.bfloat16).requires_grad_()
    kernels.moe_unpermute(y, r, h).sum().backward()
    assert h.grad.dtype is torch.bfloat16
    x = torch.randn(3, 4, H, generator=g, device=dev, requires_grad=True)
    kernels.moe_permute(x, r).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, float(topk)))


def test_refusals(dev):
    from gridbook_b200 import kernels
    r = kernels.moe_sort(torch.zeros(4, 2, dtype=torch.int32, device=dev), 3)
    x = torch.zeros(4, 16, device=dev)
    for call, kind in ((lambda: kernels.moe_sort(torch.zeros(4, device=dev, dtype=torch.int32), 3), RuntimeError),
                       (lambda: kernels.moe_sort(torch.zeros(4, 2, device=dev), 3), RuntimeError), (lambda: kernels.moe_sort(torch.zeros(4, 2, device=dev, dtype=torch.int32), 0), RuntimeError),
                       (lambda: kernels.moe_permute(x[:3], r), RuntimeError), (lambda: kernels.moe_permute(x.double(), r), TypeError),
                       (lambda: kernels.moe_unpermute(x, r), RuntimeError), (lambda: kernels.moe_unpermute(torch.zeros(8, 16, device=dev), r, torch.zeros(4, 3, device=dev)), RuntimeError),
                       (lambda: kernels.moe_permute_fp8(x[:3], r), RuntimeError), (lambda: kernels.moe_permute(x, kernels.MoESort(r.counts, r.offsets, r.order, r.place.long(), 2)), RuntimeError)):
        with pytest.raises(kind):
            call()
    a = torch.randn(4, 16, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no derivatives of their own"):
        torch.autograd.grad(kernels.moe_permute(a, r).sum(), a, create_graph=True)


def test_streams_and_graphs(dev):
    """Forward and backward on another stream, and captured: replayed on new values they give what eager calls give."""
    from gridbook_b200 import kernels
    g = _gen(dev, 6)
    T, topk, H, E = 50, 4, 256, 16
    ids = [_ids(T, topk, E, 0, g, dev) for _ in range(3)]
    xs = [torch.randn(T, H, generator=g, device=dev) for _ in range(3)]
    w = torch.rand(T, topk, generator=g, device=dev)
    d_out = torch.randn(T, H, generator=g, device=dev)

    def step(i, x, w):
        r = kernels.moe_sort(i, E)
        out = kernels.moe_unpermute(kernels.moe_permute(x, r), r, w)
        return (out, *torch.autograd.grad(out, [x, w], d_out))

    eager = [[t.detach().clone() for t in step(i, x.clone().requires_grad_(), w.clone().requires_grad_())] for i, x in zip(ids, xs)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        i, x, wg = ids[0].clone(), xs[0].clone().requires_grad_(), w.clone().requires_grad_()
        again = step(i, x, wg)
    side.synchronize()
    for p, q in zip(again, eager[0]):
        assert torch.equal(p, q)
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(i, x, wg)
    for k in (1, 2, 0):
        i.copy_(ids[k])
        with torch.no_grad():
            x.copy_(xs[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(res, eager[k]):
            assert torch.equal(p, q)


def test_expert_base_is_not_negative(dev):
    from gridbook_b200 import kernels
    for T in (4, 70000):                                                # both sorts
        ids = torch.full((T, 1), -1, dtype=torch.int64, device=dev)
        for base in (-3, 1 << 30):
            with pytest.raises(RuntimeError, match="expert_base"):
                kernels.moe_sort(ids, 8, expert_base=base)
        assert int(kernels.moe_sort(ids, 8).offsets[-1]) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_places_outside_the_rows_count_nothing(dev, dtype):
    """A sort put together by hand: places that are no row are treated as dropped pairs, a negative count as none."""
    from gridbook_b200 import kernels
    g = _gen(dev, 31)
    T, topk, H = 6, 2, 40
    x = torch.randn(T, H, generator=g, device=dev).to(dtype)
    place = torch.tensor([0, -1, 3, 12, 1, -7, 2 ** 31 - 1, 2, 4, 13, 5, -2 ** 31], dtype=torch.int32, device=dev)
    r = kernels.MoESort(None, torch.tensor([0, -9], dtype=torch.int32, device=dev), None, place, topk)
    good = [(p // topk, at) for p, at in enumerate(place.tolist()) if 0 <= at < T * topk]
    want = torch.zeros(T * topk, H, device=dev, dtype=dtype)
    for t, at in good:
        want[at] = x[t]
    none = kernels.MoESort(None, torch.tensor([0, T * topk], dtype=torch.int32, device=dev), None, place, topk)
    rows = kernels.moe_permute(x, none)
    for t, at in good:
        assert torch.equal(rows[at], x[t])
    q, s = kernels.moe_permute_fp8(x, none)
    fq, fs = kernels.fp8_quantize_blocks(x)
    for t, at in good:
        assert torch.equal(q[at].view(torch.uint8), fq[t].view(torch.uint8)) and torch.equal(s[at], fs[t])
    y = want.clone().requires_grad_()
    w = torch.ones(T, topk, device=dev, requires_grad=True)
    out = kernels.moe_unpermute(y, none, w)
    ref = torch.zeros(T, H, device=dev, dtype=torch.float64)
    for t, at in good:
        ref[t] += want[at].double()
    assert bool(((out.double() - ref).abs() <= B.HALF[dtype] * ref.abs() + 1e-6).all())
    out.sum().backward()
    for t, at in good:
        assert torch.equal(y.grad[at], torch.ones_like(y.grad[at]))
    hit = torch.zeros(T * topk, dtype=torch.bool, device=dev)
    hit[[p for p, at in enumerate(place.tolist()) if 0 <= at < T * topk]] = True
    assert not bool(w.grad.reshape(-1)[~hit].any())
    kernels.moe_permute(x, r)                                           # rows from a negative count on: all of them become zero or a token's
    torch.cuda.synchronize()


def test_rows_past_two_gigabytes(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 32)
    T, topk, H, E = 40000, 8, 7168, 16
    x = torch.zeros(T, H, dtype=torch.bfloat16, device=dev)
    x[-2:] = torch.randn(2, H, generator=g, device=dev).to(torch.bfloat16)
    ids = torch.zeros(T, topk, dtype=torch.int32, device=dev)
    ids[-2:] = E - 1                                                    # their rows come last
    r = kernels.moe_sort(ids, E)
    rows = kernels.moe_permute(x, r)
    assert rows.numel() > 2 ** 31
    assert torch.equal(rows[-2 * topk:], x[-2:].repeat_interleave(topk, 0))
    w = torch.full((T, topk), 0.125, device=dev)
    out = kernels.moe_unpermute(rows, r, w)
    assert torch.equal(out[-2:], x[-2:]) and not bool(out[-100:-2].any())
    y, wg = rows.requires_grad_(), w.requires_grad_()
    dy, dw = torch.autograd.grad(kernels.moe_unpermute(y, r, wg), [y, wg], x)
    assert torch.equal(dy[-2 * topk:], (x[-2:].float() * 0.125).to(torch.bfloat16).repeat_interleave(topk, 0))
    sq = x[-2:].double().square().sum(-1, keepdim=True)
    assert bool(((dw[-2:].double() - sq).abs() <= H * 2.0 ** -24 * sq).all())
    q, s = kernels.moe_permute_fp8(x, r)
    fq, fs = kernels.fp8_quantize_blocks(x[-2:])
    assert torch.equal(q[-2 * topk:].view(torch.uint8), fq.view(torch.uint8).repeat_interleave(topk, 0))
    assert torch.equal(s[-2 * topk:], fs.repeat_interleave(topk, 0))
