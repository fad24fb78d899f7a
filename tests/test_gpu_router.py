"""The router's choice and the experts' balance loss with their gradients: choices exactly, numbers against fp64 formulas, gradients against them
and against differences."""
import pytest
import torch

from tests.blocks import HALF

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _logits(T, E, dtype, g, dev, spread=2.0):
    return (spread * torch.randn(T, E, generator=g, device=dev)).to(dtype)


def choice(l, k, score, renormalize, scale):
    """(weights, ids) in fp64; experts at -inf are no choice."""
    l = l.double()
    ids = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :k]
    none = l.gather(1, ids) == -INF
    p = torch.softmax(l, -1) if score == "softmax" else torch.sigmoid(l)
    p = torch.where((l == -INF).all(-1, keepdim=True), torch.zeros_like(p), p)
    c = p.gather(1, ids).masked_fill(none, 0.0)
    total = c.sum(-1, keepdim=True) if renormalize else torch.ones_like(c[:, :1])
    return torch.where(total == 0, torch.zeros_like(c), c / total) * scale, ids.masked_fill(none, -1)


def slack(l):
    """Relative error of a score or a sum of scores in fp32: the argument of the exponential rounds by half a unit of itself, the
    function by two units, a sum of positive terms by one each (no more than 32 + 10 in a row), a few products."""
    l = l.double()
    fine = torch.where(torch.isfinite(l), l, torch.zeros_like(l))
    return (2.0 * (fine.amax(-1, keepdim=True) - fine.amin(-1, keepdim=True)) + 2.0 * fine.abs().amax(-1, keepdim=True) + 64.0) * U


CASES = [(1, 8, 2), (1, 1, 1), (5, 7, 3), (64, 128, 8), (300, 256, 8), (33, 129, 1), (17, 300, 6), (40, 512, 32), (9, 1000, 4), (6, 1024, 8), (3, 1025, 2), (2, 4096, 8),
         (2, 33, 32), (1000, 60, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", CASES)
def test_choice_and_gradient(dev, dtype, T, E, k):
    from gridbook_b200 import kernels
    g = _gen(dev, T + E)
    l = _logits(T, E, dtype, g, dev)
    dw = torch.randn(T, k, generator=g, device=dev)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            a = l.clone().requires_grad_()
            w, ids = kernels.moe_topk(a, k, score=score, renormalize=renormalize, scale=1.5)
            x = l.double().requires_grad_()
            want, want_ids = choice(x, k, score, renormalize, 1.5)
            assert torch.equal(ids.long(), want_ids) and ids.dtype is torch.int32 and w.dtype is torch.float32
            tol = slack(l)
            assert bool(((w.double() - want).abs() <= 2 * tol * want + 1e-37).all())
            got, = torch.autograd.grad(w, a, dw)
            ref, = torch.autograd.grad(want, x, dw.double())
            # each value is a score times a difference of two terms, each with the slack of its factors
            size = 1.5 * (dw.double().abs().amax(-1, keepdim=True)) * (torch.softmax(l.double(), -1) if score == "softmax" else torch.sigmoid(l.double()))
            if renormalize:
                size = size / choice(l, k, score, False, 1.0)[0].sum(-1, keepdim=True)
            bound = 8 * tol * size + (1 + 8 * tol) * HALF[dtype] * ref.abs() + (2.0 ** -25 if dtype is torch.float16 else 1e-37)
            assert got.dtype is dtype and bool(((got.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_expert(dev, dtype):
    from gridbook_b200 import kernels
    for E, k in ((5, 5), (128, 8), (257, 8), (1500, 8)):
        l = torch.randint(0, 3, (50, E), generator=_gen(dev, E), device=dev).to(dtype)
        l[0] = 0.0
        l[1, ::2] = -0.0                                    # zeros are alike
        l[1, 1::2] = 0.0
        ids = kernels.moe_topk(l, k)[1]
        assert torch.equal(ids.long(), choice(l + 0.0, k, "softmax", True, 1.0)[1])
        assert ids[0].tolist() == list(range(k)) and ids[1].tolist() == list(range(k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [6, 64, 700, 2000])
def test_masked_experts(dev, dtype, E):
    """-inf is never chosen, a row of it chooses nobody and has no gradient; the type's lowest value is a logit like any other."""
    from gridbook_b200 import kernels
    k = 4
    l = _logits(5, E, dtype, _gen(dev, E), dev)
    l[0] = -INF
    l[1, 2:] = -INF                                         # two are left
    l[2] = torch.finfo(dtype).min
    l[2, 5] = 0.0
    l[3, 1] = -INF
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            a = l.clone().requires_grad_()
            w, ids = kernels.moe_topk(a, k, score=score, renormalize=renormalize)
            want, want_ids = choice(l, k, score, renormalize, 1.0)
            assert torch.equal(ids.long(), want_ids)
            assert ids[0].tolist() == [-1] * k and ids[1, 2:].tolist() == [-1, -1] and ids[2].tolist() == [5, 0, 1, 2]
            rows = [0, 1, 3, 4] if dtype is torch.float32 else [0, 1, 2, 3, 4]   # slack() of the lowest fp32 value says nothing
            assert bool(((w.double() - want).abs() <= 2 * slack(l) * want + 1e-37)[rows].all())
            d, = torch.autograd.grad(w, a, torch.randn(5, k, generator=_gen(dev, 9), device=dev))
            assert bool(torch.isfinite(d).all()) and not bool(d[0].any()) and not bool(d[1, 2:].any()) and float(d[3, 1]) == 0.0
    from_sort = kernels.moe_sort(kernels.moe_topk(l, k)[1], E)
    assert int(from_sort.offsets[-1]) == 5 * k - k - 2


def test_infinities_and_nan(dev):
    from gridbook_b200 import kernels
    l = torch.zeros(3, 8, device=dev)
    l[0, 3] = float("nan")
    l[1, 6] = INF
    w, ids = kernels.moe_topk(l, 2)
    assert ids.tolist() == [[3, 0], [6, 0], [0, 1]]
    assert bool(torch.isnan(w[0]).all()) and bool(torch.isnan(w[1]).all()) and w[2].tolist() == [0.5, 0.5]
    w, ids = kernels.moe_topk(l, 2, score="sigmoid")
    assert bool(torch.isnan(w[0]).all()) and float(w[1, 0]) == pytest.approx(2 / 3, rel=1e-6)


def balance(l, ids, coef, z_coef, mask=None):
    """The loss in fp64, and the counts."""
    E = l.shape[1]
    live = torch.isfinite(l.detach().double().amax(-1)) if mask is None else mask & torch.isfinite(l.detach().double().amax(-1))
    rows, chosen = l[live], ids.long()[live].reshape(-1)
    counts = torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
    n = rows.shape[0]
    if n == 0:
        return l.sum() * 0.0, counts
    f = counts.double() / (n * ids.shape[1])
    return coef * E * (f * torch.softmax(rows, -1).mean(0)).sum() + z_coef * torch.logsumexp(rows, -1).square().mean(), counts


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", CASES + [(5000, 64, 8), (4097, 200, 2), (20000, 8, 1)])
def test_balance_loss_and_gradient(dev, dtype, T, E, k):
    from gridbook_b200 import kernels
    g = _gen(dev, T * 3 + E)
    l = _logits(T, E, dtype, g, dev)
    ids = torch.randint(-1, E + 1, (T, k), generator=g, device=dev)          # some of them nobody's
    mask = torch.rand(T, generator=g, device=dev) < 0.7
    for m in (None, mask):
        for i in (ids.int(), ids):
            a = l.clone().requires_grad_()
            loss, counts = kernels.moe_balance_loss(a, i, coef=0.5, z_coef=0.25, mask=m)
            x = l.double().requires_grad_()
            want, want_counts = balance(x, ids, 0.5, 0.25, m)
            assert loss.shape == () and loss.dtype is torch.float32 and counts.dtype is torch.int32 and torch.equal(counts.long(), want_counts)
            tol = float(slack(l).max()) + (T // 4000 + 64) * U               # sums of positive terms over tokens: a group's own, then the groups'
            assert abs(float(loss) - float(want)) <= 2 * tol * float(want)
            got, = torch.autograd.grad(loss, a, torch.tensor(3.0, device=dev))
            ref, = torch.autograd.grad(want, x, torch.tensor(3.0, dtype=torch.double, device=dev))
            n = T if m is None else max(int(m.sum()), 1)
            p = torch.softmax(l.double(), -1)
            f = want_counts.double() / (n * k)
            size = 3.0 / n * p * (0.5 * E * (f + (f * p).sum(-1, keepdim=True)) + 0.5 * torch.logsumexp(l.double(), -1, keepdim=True).abs())
            bound = 8 * tol * size + (1 + 8 * tol) * HALF[dtype] * ref.abs() + (2.0 ** -25 if dtype is torch.float16 else 1e-37)
            assert bool(((got.double() - ref).abs() <= bound).all())
            if m is not None:
                assert not bool(got[~m].any())


def test_balance_of_nothing(dev):
    from gridbook_b200 import kernels
    for l, ids, mask in ((torch.empty(0, 6, device=dev), torch.empty(0, 2, dtype=torch.int32, device=dev), None),
                         (torch.zeros(4, 6, device=dev), torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.bool, device=dev)),
                         (torch.full((4, 6), -INF, device=dev), torch.zeros(4, 2, dtype=torch.int32, device=dev), None)):
        l.requires_grad_()
        loss, counts = kernels.moe_balance_loss(l, ids, coef=1.0, z_coef=1.0, mask=mask)
        assert float(loss) == 0.0 and counts.tolist() == [0] * 6
        d, = torch.autograd.grad(loss, l)
        assert d.shape == l.shape and not bool(d.any())
    l = torch.zeros(3, 4, device=dev)
    l[1] = -INF                                             # counts as masked: what it chose too
    loss, counts = kernels.moe_balance_loss(l, torch.tensor([[0], [1], [2]], device=dev), coef=1.0)
    assert counts.tolist() == [1, 0, 1, 0] and float(loss) == pytest.approx(1.0, rel=1e-6)


def test_even_routing_costs_the_coefficient(dev):
    from gridbook_b200 import kernels
    ids = torch.arange(64, device=dev).view(16, 4) % 8
    loss, counts = kernels.moe_balance_loss(torch.zeros(16, 8, device=dev), ids, coef=0.25)
    assert float(loss) == 0.25 and counts.tolist() == [8] * 8


def test_gradients_against_differences(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 5)
    l = _logits(6, 10, torch.float32, g, dev)
    ids = torch.randint(0, 10, (6, 2), generator=g, device=dev)
    dw = torch.randn(6, 2, generator=g, device=dev)
    step = 2.0 ** -7
    for f in (lambda x: (kernels.moe_topk(x, 2)[0] * dw).sum(), lambda x: (kernels.moe_topk(x, 2, score="sigmoid", renormalize=False)[0] * dw).sum(),
              lambda x: (kernels.moe_topk(x, 2, renormalize=False)[0] * dw).sum(), lambda x: kernels.moe_balance_loss(x, ids, coef=1.0, z_coef=0.5)[0]):
        x = l.clone().requires_grad_()
        got, = torch.autograd.grad(f(x), x)
        for t, e in ((0, 0), (2, 7), (5, 9), (3, int(l[3].argmax()))):
            up, down = l.clone(), l.clone()
            up[t, e] += step
            down[t, e] -= step
            if not torch.equal(kernels.moe_topk(up, 2)[1], kernels.moe_topk(down, 2)[1]):
                continue
            # a third derivative of order one times step^2 / 6, and the rounding of sums of a few units over the step
            assert abs(float((f(up) - f(down)) / (2 * step)) - float(got[t, e])) < 4 * step ** 2 + 64 * U * 8 / step


def test_strides_types_and_refusals(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 7)
    base = torch.randn(30, 70, generator=g, device=dev)
    ids = torch.randint(0, 16, (30, 2), generator=g, device=dev)
    for l in (base[:, 3:19], base[:, 4:20], base.t()[:30, :16], base[:1, :16].expand(30, 16), base[::2, :16]):
        w, i = kernels.moe_topk(l, 3)
        w2, i2 = kernels.moe_topk(l.contiguous(), 3)
        assert torch.equal(w, w2) and torch.equal(i, i2)
        rows = ids[:l.shape[0]]
        one, two = kernels.moe_balance_loss(l, rows.short()), kernels.moe_balance_loss(l.contiguous(), rows.t().contiguous().t())
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    far = ids.clone()
    far[0] = (1 << 32) + 3                                  # nobody's, whatever the low half says
    assert int(kernels.moe_balance_loss(base[:, :16], far)[1].sum()) == 58
    l = base[:, :16]
    for call, kind in ((lambda: kernels.moe_topk(l, 0), RuntimeError), (lambda: kernels.moe_topk(l, 17), RuntimeError), (lambda: kernels.moe_topk(l[0], 2), RuntimeError),
                       (lambda: kernels.moe_topk(l.double(), 2), TypeError), (lambda: kernels.moe_topk(l, 2, score="relu"), RuntimeError),
                       (lambda: kernels.moe_balance_loss(l, ids[:4]), RuntimeError), (lambda: kernels.moe_balance_loss(l, ids.float()), RuntimeError),
                       (lambda: kernels.moe_balance_loss(l, ids, mask=torch.ones(30, device=dev)), RuntimeError),
                       (lambda: kernels.moe_balance_loss(l, ids, mask=torch.ones(3, dtype=torch.bool, device=dev)), RuntimeError),
                       (lambda: kernels.moe_balance_loss(l, ids.cpu()), RuntimeError)):
        with pytest.raises(kind):
            call()
    a = l.clone().requires_grad_()
    for out in (kernels.moe_topk(a, 2)[0].sum(), kernels.moe_balance_loss(a, ids)[0]):
        with pytest.raises(RuntimeError, match="no derivatives of their own"):
            torch.autograd.grad(out, a, create_graph=True)
    w, i = kernels.moe_topk(a, 2)
    i.add_(1)                                               # what the backward pass reads was changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()
    assert kernels.moe_topk(torch.empty(0, 8, device=dev), 2)[0].shape == (0, 2)


def test_streams_and_graphs(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 11)
    ls = [_logits(400, 96, torch.float32, g, dev) for _ in range(3)]
    dw = torch.randn(400, 4, generator=g, device=dev)

    def step(l):
        w, ids = kernels.moe_topk(l, 4)
        loss, counts = kernels.moe_balance_loss(l, ids, coef=1.0, z_coef=0.1)
        return (w.detach(), ids, loss.detach(), counts, *torch.autograd.grad([w, loss], [l], [dw, torch.ones_like(loss)]))

    eager = [[t.clone() for t in step(l.clone().requires_grad_())] for l in ls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        l = ls[0].clone().requires_grad_()
        again = step(l)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(again, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(l)
    for k in (1, 2, 0):
        with torch.no_grad():
            l.copy_(ls[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, eager[k]))
