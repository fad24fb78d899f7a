"""16-bit linears with bias, activation and residual, and their gradients, against fp64: every activation and epilogue, single rows, ragged
sizes on both kernels, split contractions, strides, streams and graphs."""
import math

import pytest
import torch

from tests.blocks import HALF

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
F = torch.nn.functional
FN = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}
STEEPEST = 1.13            # largest slope of any of them (gelu's, at sqrt 2)
BEND = 0.8                 # largest second derivative (gelu's, 2 / sqrt(2 pi), and the others' below it); relu's none, but at zero
ADD = 2.0 ** -23           # a sum on the tensor cores: each addition off by at most a whole unit (how they round is not specified)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _inputs(M, N, K, dtype, bias, residual, g, dev):
    def n(*shape):
        return torch.randn(*shape, generator=g, device=dev)
    return n(M, K).to(dtype), (n(N, K) * (1.5 / math.sqrt(K))).to(dtype), n(N).to(dtype) if bias else None, n(M, N).to(dtype) if residual else None


def _low(dtype):
    return 2.0 ** -25 if dtype is HF else 1e-38


def product(x, w, b):
    """z in fp64 and what its fp32 sums may be off by: K additions and the bias."""
    x, w = x.double(), w.double()
    z, size = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    return z, (x.shape[-1] + 2) * ADD * size


def check(got, ref, err, dtype, name):
    tol = err + (1 + 2.0 ** -8) * HALF[dtype] * ref.abs() + _low(dtype)
    off = (got.double() - ref).abs() - tol
    assert got.dtype is dtype and bool(torch.isfinite(got).all()) and float(off.max()) <= 0.0, \
        f"{name}: {int((off > 0).sum())} of {off.numel()} off, by up to {float(off.max()):.3e}"


def check_forward(y, x, w, b, act, r, name=""):
    z, ez = product(x, w, b)
    ref = FN[act](z)
    # the activation in fp32: a few units of its argument; the residual's addition
    err = STEEPEST * ez + 16 * 2.0 ** -23 * (z.abs() + ez)
    if r is not None:
        ref = ref + r.double()
        err = err + 2.0 ** -23 * (ref.abs() + r.double().abs())
    check(y, ref, err * (1 + 2.0 ** -8), y.dtype, f"y {name}")


def check_grads(got, x, w, b, act, dy, name=""):
    """``got``: gradients of x, w, b.  z is read back rounded to the type: the slope moves by its second derivative times that; dz is
    rounded to the type for the products (where there is an activation)."""
    dtype = x.dtype
    z, ez = product(x, w, b)
    ez = ez + HALF[dtype] * z.abs() + _low(dtype) if act else 0 * ez
    zl = z.clone().requires_grad_()
    slope, = torch.autograd.grad(FN[act](zl).sum(), zl)
    g = dy.double()
    dz = g * slope
    e = g.abs() * (BEND * ez + 2.0 ** -20 if act not in (None, "relu") else (z.abs() <= ez).double() if act == "relu" else 0 * ez)
    M, N, K = z.shape[0], z.shape[1], x.shape[1]
    if got[2] is not None:
        check(got[2], dz.sum(0), e.sum(0) + (M + 4) * 2.0 ** -24 * dz.abs().sum(0), dtype, f"db {name}")
    if act:
        e = e + HALF[dtype] * (dz.abs() + e) + _low(dtype)
    xa, wa, xd, wd = x.double().abs(), w.double().abs(), x.double(), w.double()
    size = dz.abs() + e
    if got[0] is not None:
        check(got[0], dz @ wd, e @ wa + (N + 2) * ADD * (size @ wa), dtype, f"dx {name}")
    if got[1] is not None:
        check(got[1], dz.T @ xd, e.T @ xa + (M + 18) * ADD * (size.T @ xa), dtype, f"dw {name}")


SHAPES = [(1, 256, 256), (2, 300, 264), (4, 129, 1024), (1, 130, 8192), (1, 4096, 4096), (3, 1, 8), (7, 1000, 264), (16, 640, 1024), (130, 129, 72), (192, 512, 2048), (200, 1024, 256), (256, 8, 64), (257, 520, 520),
          (333, 1111, 1000), (700, 2304, 512), (1100, 1001, 136), (1500, 384, 64), (2100, 776, 200), (513, 16384, 128), (1024, 2048, 4096)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_forward(dev, dtype, M, N, K):
    from gridbook_b200 import kernels
    g = _gen(dev, M + N + K)
    for act, bias, residual in ((None, False, False), ("gelu", True, False), ("silu", True, True), (None, True, True), ("relu", False, True)):
        x, w, b, r = _inputs(M, N, K, dtype, bias, residual, g, dev)
        y = kernels.linear_act(x, w, b, activation=act, residual=r)
        assert y.shape == (M, N)
        check_forward(y, x, w, b, act, r, f"{act} {bias} {residual}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gradients(dev, dtype, M, N, K):
    from gridbook_b200 import kernels
    g = _gen(dev, 3 * M + N + K)
    for act, bias, residual in (("gelu_tanh", True, True), (None, True, False), ("silu", False, False), ("relu", True, True), ("gelu", False, True), (None, False, False)):
        x, w, b, r = _inputs(M, N, K, dtype, bias, residual, g, dev)
        leaves = [t.clone().requires_grad_() if t is not None else None for t in (x, w, b, r)]
        y = kernels.linear_act(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
        check_forward(y, x, w, b, act, r, f"{act} {bias} {residual}")
        dy = torch.randn(M, N, generator=g, device=dev).to(dtype)
        got = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
        got = [next(got) if t is not None else None for t in leaves]
        check_grads(got, x, w, b, act, dy, f"{act} {bias} {residual}")
        if residual:
            assert torch.equal(got[3], dy)


@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(dev, act):
    """Arguments from far below to far above, exactly representable: one input of one, weights that are the arguments."""
    from gridbook_b200 import kernels
    for dtype in (BF, HF):
        big = 3e4 if dtype is HF else 1e30
        z = torch.cat([torch.linspace(-12, 12, 2000, device=dev), torch.tensor([0.0, -0.0, big, -big, 1e-6, -1e-6, 100.0, -100.0], device=dev)]).to(dtype)
        N = z.numel()
        x = torch.zeros(1, 8, dtype=dtype, device=dev)
        x[0, 0] = 1.0
        for M in (1, 300):                                    # both kernels
            w = torch.zeros(N, 8, dtype=dtype, device=dev)
            w[:, 0] = z
            lx, lw, lb = x.expand(M, 8).contiguous().requires_grad_(), w.requires_grad_(), torch.zeros(N, dtype=dtype, device=dev, requires_grad=True)
            y = kernels.linear_act(lx, lw, lb, activation=act)
            ref = FN[act](z.double())
            tol = HALF[dtype] * ref.abs() * (1 + 2.0 ** -8) + 16 * 2.0 ** -23 * z.double().abs().clamp(max=16) + _low(dtype)
            assert bool(((y.double() - ref).abs() <= tol).all())
            db, = torch.autograd.grad(y, lb, torch.full_like(y, 1.0 / 256))
            zl = z.double().requires_grad_()
            slope, = torch.autograd.grad(FN[act](zl).sum(), zl)
            want = slope * M / 256
            keep = z != 0 if act == "relu" else torch.ones_like(z, dtype=torch.bool)   # (torch takes relu's slope at zero as zero too)
            assert bool(((db.double() - want).abs() <= HALF[dtype] * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -18 * M / 256 + _low(dtype))[keep].all())


def test_what_is_not_asked_for(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 4)
    for M, N, K in ((40, 264, 136), (300, 1001, 64)):
        x, w, b, r = _inputs(M, N, K, BF, True, True, g, dev)
        dy = torch.randn(M, N, generator=g, device=dev).to(BF)
        for act in (None, "gelu"):
            for need in ((0,), (1,), (2,), (3,), (0, 2), (1, 3)):
                t = [v.clone().requires_grad_(i in need) for i, v in enumerate((x, w, b, r))]
                y = kernels.linear_act(t[0], t[1], t[2], activation=act, residual=t[3])
                grads = dict(zip(need, torch.autograd.grad(y, [t[i] for i in need], dy)))
                check_grads([grads.get(i) for i in range(3)], x, w, b, act, dy, f"{act} {need}")
                if 3 in need:
                    assert torch.equal(grads[3], dy)


def test_infinities_and_nan_stay_in_their_rows(dev):
    from gridbook_b200 import kernels
    for M in (4, 300):
        x = torch.zeros(M, 64, dtype=BF, device=dev)
        x[1, 3], x[2, 5] = float("nan"), float("inf")
        w = torch.ones(96, 64, dtype=BF, device=dev)
        for act in ACTS:
            y = kernels.linear_act(x, w, activation=act)
            assert bool(torch.isnan(y[1]).all()) and bool((y[2] == float("inf")).all()) and not bool(y[0].any()) and not bool(y[3:].any())


def test_shapes_strides_and_rows_elsewhere(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 6)
    base, w = torch.randn(48, 320, generator=g, device=dev).to(BF), (torch.randn(200, 256, generator=g, device=dev) / 16).to(BF)
    res = torch.randn(48, 420, generator=g, device=dev).to(BF)
    b = torch.randn(400, generator=g, device=dev).to(BF)
    for x in (base[:, 8:264], base[:, 3:259], base[:, 4:260], base[::2, :256], base.t()[:256].t()):
        for r in (res[:, 16:216], res[:, 7:207], res.t()[:200].t()):
            r = r[:x.shape[0]]
            got = kernels.linear_act(x, w, b[::2], activation="silu", residual=r)
            want = kernels.linear_act(x.contiguous(), w.contiguous(), b[::2].contiguous(), activation="silu", residual=r.contiguous())
            assert torch.equal(got, want)
    flat = torch.randn(200 * 256 + 8, generator=g, device=dev).to(BF)
    for wt in (w.t().contiguous().t(), flat[1:1 + 200 * 256].view(200, 256)):
        x = base[:, :256].contiguous().requires_grad_()
        got, want = kernels.linear_act(x, wt), kernels.linear_act(x, wt.clone(memory_format=torch.contiguous_format))
        assert torch.equal(got, want)
        assert torch.equal(torch.autograd.grad(got.sum(), x)[0], torch.autograd.grad(want.sum(), x)[0])
    x3 = base[:, :256].reshape(2, 3, 8, 256).clone().requires_grad_()
    y = kernels.linear_act(x3, w, residual=res[:, :200].reshape(2, 3, 8, 200))
    assert y.shape == (2, 3, 8, 200)
    dx, = torch.autograd.grad(y, x3, torch.ones((), dtype=BF, device=dev).expand_as(y))
    assert dx.shape == x3.shape
    assert kernels.linear_act(base[0, :256], w).shape == (200,)
    x0, w0 = torch.empty(0, 256, dtype=BF, device=dev, requires_grad=True), w.clone().requires_grad_()
    y = kernels.linear_act(x0, w0, b[:200].clone().requires_grad_(), activation="gelu")
    dx, dw = torch.autograd.grad(y, [x0, w0], torch.empty_like(y))
    assert y.shape == (0, 200) and dx.shape == (0, 256) and not bool(dw.any())


def test_refusals(dev):
    from gridbook_b200 import kernels
    x, w, b, r = _inputs(6, 40, 64, BF, True, True, _gen(dev, 7), dev)
    for call, kind in ((lambda: kernels.linear_act(x.float(), w.float()), TypeError), (lambda: kernels.linear_act(x, w.half()), RuntimeError),
                       (lambda: kernels.linear_act(x, w[:, :32]), RuntimeError), (lambda: kernels.linear_act(x[:, :60], w[:, :60]), RuntimeError),
                       (lambda: kernels.linear_act(x, w, b[:3]), RuntimeError), (lambda: kernels.linear_act(x, w, b.float()), RuntimeError),
                       (lambda: kernels.linear_act(x, w, b, residual=r[:1]), RuntimeError), (lambda: kernels.linear_act(x, w, b, residual=r.float()), RuntimeError),
                       (lambda: kernels.linear_act(x, w.cpu()), RuntimeError), (lambda: kernels.linear_act(x, w[0]), RuntimeError),
                       (lambda: kernels.linear_act(x, w, activation="selu"), ValueError)):
        with pytest.raises(kind):
            call()
    a = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no derivatives of their own"):
        torch.autograd.grad(kernels.linear_act(a, w).sum(), a, create_graph=True)
    a, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = kernels.linear_act(a, wg)
    with torch.no_grad():
        wg.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_against_differences(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 8)
    x, w, b, _ = _inputs(5, 16, 24, HF, True, False, g, dev)
    dy = torch.randn(5, 16, generator=g, device=dev).to(HF)
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        got = torch.autograd.grad(kernels.linear_act(*leaves, activation=act), leaves, dy)
        step = 2.0 ** -3
        for i, at in ((0, (1, 5)), (1, (3, 20)), (2, (7,))):
            up, down = [t.clone() for t in (x, w, b)], [t.clone() for t in (x, w, b)]
            up[i][at] += step
            down[i][at] -= step
            moved = float(up[i][at] - down[i][at])
            change = ((kernels.linear_act(*up, activation=act).double() - kernels.linear_act(*down, activation=act).double()) * dy.double()).sum() / moved
            # up to 16 outputs moved: each rounded to fp16 (|y| to about 8) on both sides; third derivatives of order one
            assert abs(float(change) - float(got[i][at])) < 16 * 8 * HALF[HF] * 2 / moved + 16 * 4 * step ** 2 + 0.01


def test_streams_and_graphs(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 9)
    for M, N, K in ((24, 512, 256), (400, 640, 512)):
        sets = [_inputs(M, N, K, BF, True, True, g, dev) for _ in range(3)]
        dy = torch.randn(M, N, generator=g, device=dev).to(BF)

        def step(t):
            y = kernels.linear_act(t[0], t[1], t[2], activation="gelu", residual=t[3])
            return (y.detach(), *torch.autograd.grad(y, t, dy))
        eager = [[v.clone() for v in step([v.clone().requires_grad_() for v in t])] for t in sets]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            t = [v.clone().requires_grad_() for v in sets[0]]
            again = step(t)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(again, eager[0]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = step(t)
        for k in (1, 2, 0):
            with torch.no_grad():
                for a, c in zip(t, sets[k]):
                    a.copy_(c)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(res, eager[k]))


def test_two_streams_at_once(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 10)
    a, b = _inputs(900, 2048, 1024, BF, True, True, g, dev), _inputs(16, 4096, 2048, BF, True, True, g, dev)
    want = [kernels.linear_act(*t[:3], activation="silu", residual=t[3]) for t in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            outs.append((0, kernels.linear_act(*a[:3], activation="silu", residual=a[3])))
        with torch.cuda.stream(s2):
            outs.append((1, kernels.linear_act(*b[:3], activation="silu", residual=b[3])))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in outs)


def test_past_two_to_the_31_values(dev):
    """Rows of the result behind its 2^31st value, on the kernel of many rows."""
    from gridbook_b200 import kernels
    g = _gen(dev, 11)
    M, N, K = 66000, 33000, 64
    x, w = torch.randn(M, K, generator=g, device=dev).to(BF), (torch.randn(N, K, generator=g, device=dev) / 8).to(BF)
    b = torch.randn(N, generator=g, device=dev).to(BF)
    r = torch.ones(1, 1, dtype=BF, device=dev).expand(M, N).contiguous()
    y = kernels.linear_act(x, w, b, activation="relu", residual=r)
    assert y.numel() > 2 ** 31
    check_forward(y[-40:], x[-40:], w, b, "relu", r[-40:])
    check_forward(y[:40], x[:40], w, b, "relu", r[:40])


@pytest.mark.parametrize("M,N,K,dtype", [(256, 16384, 7232, HF), (256, 8200, 7232, BF), (251, 8195, 4096, HF), (40, 16384, 8192, BF)])
def test_the_step_of_a_relu_falls_where_z_crosses_zero(dev, M, N, K, dtype):
    """With ones as the gradient the bias' gradient counts a column's positive values, exactly up to 256 of them.  Values near zero are summed
    up in fp32: some 2^-25 sqrt(K / 8) / sqrt(32) of z's spread off (K / 64 additions in each of two chains of a lane, whose sums are
    sqrt(32) smaller; the sums over the lanes are less), so that less than one in ten million changes its sign; three of 4 million are allowed.  Sums
    that drop bits at each step of the tensor cores turn a few in a million.  Some columns and rows are small as a whole, one column is
    zero throughout."""
    from gridbook_b200 import kernels
    g = _gen(dev, 70 + K % 64 + M)
    x, w, b, _ = _inputs(M, N, K, dtype, True, False, g, dev)
    w[3::64] *= 2.0 ** -9
    b[3::64] *= 2.0 ** -9
    w[7], b[7] = 0.0, 0.0
    x[5] *= 2.0 ** -6
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    y = kernels.linear_act(x, w, b, activation="relu")
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    with torch.no_grad():
        turned = 0
        for n in range(0, N, 2048):
            z = x.double() @ w[n:n + 2048].double().T + b[n:n + 2048].double()
            low = (z.abs() < _low(dtype)) if dtype is HF else torch.zeros_like(z, dtype=torch.bool)     # fp16 keeps no smaller z
            off = (db[n:n + 2048].double() - (z > 0).double().sum(0)).abs()
            turned += int((off - low.sum(0)).clamp(min=0).sum())
    assert float(db[7]) == 0.0 and turned <= 3, turned
