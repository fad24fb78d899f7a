"""The norms behind and in front of a block with their gradients, against fp64 formulas: values, gradients of everything, gates of every form, types,
odd and long rows, blocks of E4M3, masks of broadcast inputs."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = B.HALF
TYPES = [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)]
U = 2.0 ** -24
EPS = 1e-5
A, BR = 0.75, 1.25                                        # scales of the residual and of the branch
SHAPES = [(1, 8), (1, 5120), (3, 64), (5, 1001), (40, 2048), (7, 2056), (130, 768), (2, 8192), (3, 8200), (2, 16384), (2, 20000), (1500, 72), (300, 33)]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _inputs(T, H, dtype, stream, gate, post, g, dev, weights=None):
    def n(*shape):
        return torch.randn(*shape, generator=g, device=dev)
    y, r = (3.0 * n(T, H)).to(dtype), (2.0 * n(T, H)).to(stream)
    w, pw = ((1.0 + 0.3 * n(H)).to(weights or dtype) for _ in range(2))
    shape = {"none": None, "channel": (H,), "full": (T, H)}[gate]
    return y, r, w, pw if post else None, None if shape is None else n(*shape).to(dtype)


def rms(v):
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)


def depth(H):
    """Most fp32 additions that a value of a sum over a row goes through, and the rounding of what is added: a thread's own columns (sixteen,
    or every 256th), two butterflies over a warp."""
    return 28 + max(16, H // 256 + 1)


def er(H):
    """Relative error of 1 / rms: half that of a mean of squares (each square's rounding, the sum, the mean, eps), two units of the root."""
    return (0.5 * (depth(H) + 3) + 4) * U


def stream_of(y, r, pw, gate, offset=0.0):
    """The stream in fp64 and the size of what the error is relative to."""
    u = y.double() if pw is None else rms(y.double()) * (offset + pw.double())
    b = BR * (u if gate is None else gate.double() * u)
    return A * r.double() + b, A * r.double().abs() + b.abs()


def grads(s, y, w, pw, gate, dh, ds, offset=0.0, scales=(A, BR), eps=EPS):
    """(gradients, what fp32 may be off by) in fp64, the stream as it is stored: of y, residual, weight, post weight, and of the gate for each row."""
    H = s.shape[-1]
    res, br = scales
    s, y, dh, ds = (t.double() for t in (s, y, dh, ds))
    c = (depth(H) + 24) * U                               # of a sum over a row, and of the few products around it
    rs = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    xh = s * rs
    k = dh * (offset + w.double())
    m1, m1s = (k * xh).mean(-1, keepdim=True), (k * xh).abs().mean(-1, keepdim=True)
    dx = ds + rs * (k - xh * m1)
    e_dx = c * (ds.abs() + rs * (k.abs() + 2 * xh.abs() * m1s)) * 2
    g = br if gate is None else br * gate.double()
    ga = abs(g) if gate is None else g.abs()
    du, e_du = g * dx, ga * e_dx + 2 * U * (g * dx).abs()
    if pw is None:
        u, dy, e_dy, dpw, e_dpw = y, du, e_du, None, None
    else:
        p = offset + pw.double()
        rp = 1.0 / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        yh = y * rp
        u, t, e_t = yh * p, du * p, e_du * p.abs() + U * (du * p).abs()
        m2, m2s = (t * yh).mean(-1, keepdim=True), (t * yh).abs().mean(-1, keepdim=True)
        dy = rp * (t - yh * m2)
        e_dy = rp * (e_t + yh.abs() * (e_t * yh.abs()).mean(-1, keepdim=True)) + 2 * c * rp * (t.abs() + 2 * yh.abs() * m2s)
        dpw, e_dpw = du * yh, e_du * yh.abs() + 2 * c * (du * yh).abs()
    dg, e_dg = br * dx * u, br * e_dx * u.abs() + 2 * c * (br * dx * u).abs()
    return {"y": (dy, e_dy), "r": (res * dx, res * e_dx + U * (res * dx).abs()), "w": (dh * xh, 2 * c * (dh * xh).abs()), "pw": (dpw, e_dpw), "g": (dg, e_dg)}


def near(got, ref, err, name):
    tol = err + (1.0 + 2.0 ** -8) * HALF[got.dtype] * ref.abs() + (2.0 ** -25 if got.dtype is HF else 1e-38)
    off = (got.double() - ref).abs() - tol
    assert bool(torch.isfinite(got).all()) and float(off.max()) <= 0.0, f"{name}: {int((off > 0).sum())} of {off.numel()} off, by up to {float(off.max()):.3e}"


def summed(pair, T):
    """Rows' sums: every term's error, and one rounding of a partial sum a row."""
    v, e = pair
    return v.sum(0), e.sum(0) + (T + 40) * U * v.abs().sum(0)


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("T,H", SHAPES)
def test_values_and_gradients(dev, dtype, stream, T, H):
    from gridbook_b200 import kernels
    g = _gen(dev, T * 7 + H)
    for gate, post, offset in (("channel", True, 0.0), ("none", False, 0.0), ("full", True, 1.0), ("channel", False, 0.0), ("none", True, 1.0), ("full", False, 0.0), ("none", True, 0.0)):
        y, r, w, pw, gt = _inputs(T, H, dtype, stream, gate, post, g, dev)
        leaves = {k: v.clone().requires_grad_() for k, v in dict(y=y, r=r, w=w, pw=pw, g=gt).items() if v is not None}
        h, s = kernels.residual_norm(leaves["y"], leaves["r"], leaves["w"], post_weight=leaves.get("pw"), gate=leaves.get("g"), residual_scale=A, branch_scale=BR,
                                     eps=EPS, weight_offset=offset)
        assert h.dtype is dtype and s.dtype is stream and h.shape == s.shape == y.shape
        want, size = stream_of(y, r, pw, gt, offset)
        near(s, want, (er(H) + 8 * U) * size, "stream")
        near(h, rms(s.double()) * (offset + w.double()), (er(H) + 8 * U) * (rms(s.double()) * (offset + w.double())).abs(), "h")
        dh, ds = torch.randn(T, H, generator=g, device=dev).to(dtype), torch.randn(T, H, generator=g, device=dev).to(stream)
        ref = grads(s.detach(), y, w, pw, gt, dh, ds, offset)
        if gate != "full":
            ref["g"] = summed(ref["g"], T)
        ref["w"] = summed(ref["w"], T)
        if post:
            ref["pw"] = summed(ref["pw"], T)
        got = torch.autograd.grad([h, s], list(leaves.values()), [dh, ds])
        for name, t, leaf in zip(leaves, got, leaves.values()):
            assert t.dtype is leaf.dtype and t.shape == leaf.shape
            near(t, *ref[name], f"{gate} {post}: {name}")


@pytest.mark.parametrize("H", [768, 1001])
def test_gates_for_groups_of_rows(dev, H):
    """One gate for each sequence of a batch, and other leading sizes; what the gate is shared by adds up in its gradient."""
    from gridbook_b200 import kernels
    g = _gen(dev, H)
    for lead, shape in (((4, 33), (4, 1, H)), ((4, 33), (1, 1, H)), ((4, 33), (4, 33, H)), ((2, 3, 5), (2, 1, 1, H)), ((2, 3, 5), (2, 3, 1, H)), ((1, 7), (7, H)),
                        ((300, 3), (300, 1, H)), ((2000, 2), (2000, 1, H)), ((1500, 3), (1500, 1, H)), ((6, 1), (6, 1, H)), ((5, 200), (H,))):
        T = torch.Size(lead).numel()
        y, r, w, pw, _ = _inputs(T, H, BF, F32, "none", True, g, dev)
        gt = torch.randn(*shape, generator=g, device=dev).to(BF)
        full = gt.expand(*lead, H).reshape(T, H)
        leaf = gt.clone().requires_grad_()
        ly = y.view(*lead, H).requires_grad_()
        h, s = kernels.residual_norm(ly, r.view(*lead, H), w, post_weight=pw, gate=leaf, residual_scale=A, branch_scale=BR, eps=EPS)
        h2, s2 = kernels.residual_norm(y, r, w, post_weight=pw, gate=full.contiguous(), residual_scale=A, branch_scale=BR, eps=EPS)
        assert torch.equal(h.view(T, H), h2) and torch.equal(s.view(T, H), s2)
        dh, ds = torch.randn(T, H, generator=g, device=dev).to(BF), torch.randn(T, H, generator=g, device=dev)
        got, dy = torch.autograd.grad([h, s], [leaf, ly], [dh.view(*lead, H), ds.view(*lead, H)])
        ref = grads(s.detach().view(T, H), y, w, pw, full, dh, ds)
        near(dy.view(T, H), *ref["y"], "y")
        v, e = ref["g"]
        v, e = (t.view(*lead, H).sum_to_size(shape) for t in (v, e + 2 * T * U * v.abs()))
        near(got, v, e, str(shape))


def test_what_is_not_asked_for(dev):
    """Single gradients, gradients of one of the two results, no weight; and a result that nobody uses."""
    from gridbook_b200 import kernels
    g = _gen(dev, 3)
    for T, H in ((9, 256), (9, 251)):
        y, r, w, pw, gt = _inputs(T, H, F32, F32, "channel", True, g, dev)
        dh, ds = torch.randn(T, H, generator=g, device=dev), torch.randn(T, H, generator=g, device=dev)
        zero = torch.zeros_like(dh)
        names = ("y", "r", "w", "pw", "g")

        def run(need, use_h, use_s):
            t = [v.clone().requires_grad_(k in need) for k, v in zip(names, (y, r, w, pw, gt))]
            h, s = kernels.residual_norm(t[0], t[1], t[2], post_weight=t[3], gate=t[4], residual_scale=A, branch_scale=BR, eps=EPS)
            outs = ([h] if use_h else []) + ([s] if use_s else [])
            return s, torch.autograd.grad(outs, [v for v in t if v.requires_grad], ([dh] if use_h else []) + ([ds] if use_s else []))
        for need in [(n,) for n in names] + [names, ("y", "g"), ("r", "pw")]:
            for use_h, use_s in ((True, True), (True, False), (False, True)):
                s, got = run(need, use_h, use_s)
                ref = grads(s.detach(), y, w, pw, gt, dh if use_h else zero, ds if use_s else zero)
                for n, t in zip([n for n in names if n in need], got):
                    near(t, *(summed(ref[n], T) if n in ("w", "pw", "g") else ref[n]), f"{need} {n}")
        plain = y.clone().requires_grad_()                                   # without a norm behind the block its rows are not read again
        h, s = kernels.residual_norm(plain, r, w, eps=EPS)
        with torch.no_grad():
            plain.zero_()
        dy, = torch.autograd.grad([h, s], [plain], [dh, ds])
        near(dy, *grads(s.detach(), y, w, None, None, dh, ds, scales=(1.0, 1.0))["y"], "y, not kept")
        h, s = kernels.residual_norm(y, r, eps=EPS)                          # neither weights nor scales nor a gate
        want = y.double() + r.double()
        near(s, want, 4 * U * (y.double().abs() + r.double().abs()), "stream")
        near(h, rms(s.double()), (er(H) + 8 * U) * rms(s.double()).abs(), "h")
        assert not h.requires_grad


@pytest.mark.parametrize("dtype,weights", [(BF, F32), (F32, BF), (HF, BF)])
def test_weights_of_another_type(dev, dtype, weights):
    from gridbook_b200 import kernels
    g = _gen(dev, 21)
    for T, H in ((50, 512), (5, 77)):
        y, r, w, pw, gt = _inputs(T, H, dtype, F32, "channel", True, g, dev, weights)
        w, pw = w.requires_grad_(), pw.requires_grad_()
        h, s = kernels.residual_norm(y, r, w, post_weight=pw, gate=gt, residual_scale=A, branch_scale=BR, eps=EPS)
        dh, ds = torch.randn(T, H, generator=g, device=dev).to(dtype), torch.randn(T, H, generator=g, device=dev)
        dw, dpw = torch.autograd.grad([h, s], [w, pw], [dh, ds])
        ref = grads(s.detach(), y, w.detach(), pw.detach(), gt, dh, ds)
        assert dw.dtype is dpw.dtype is weights
        near(dw, *summed(ref["w"], T), "w")
        near(dpw, *summed(ref["pw"], T), "pw")


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("T,H", [(1, 128), (1, 5120), (5, 1001), (130, 768), (3, 200), (2, 7168), (2, 16384), (1, 20000), (400, 72)])
def test_blocks_of_e4m3(dev, dtype, stream, T, H):
    """Block scales to the error of h; values to a half step of E4M3 of h over the scale that was given, and what h may be off by."""
    from gridbook_b200 import kernels
    g = _gen(dev, T + H)
    for gate, post in (("channel", True), ("none", False), ("full", True)):
        y, r, w, pw, gt = _inputs(T, H, dtype, stream, gate, post, g, dev)
        for rule in ("recip", "div"):
            q, scale, s = kernels.residual_norm_fp8(y, r, w, post_weight=pw, gate=gt, residual_scale=A, branch_scale=BR, eps=EPS, scale_rule=rule)
            assert torch.equal(s, kernels.residual_norm(y, r, w, post_weight=pw, gate=gt, residual_scale=A, branch_scale=BR, eps=EPS)[1])
            want, size = stream_of(y, r, pw, gt)
            x_off = (er(H) + 8 * U) * size
            inv = 1.0 / torch.sqrt(want.square().mean(-1, keepdim=True) + EPS)
            h = want * inv * w.double()
            # the row's norm moves by what the stream is off by, in the mean
            off = (x_off * inv + want.abs() * inv * (er(H) + (x_off * want.abs()).mean(-1, keepdim=True) * inv.square()) + 4 * U * h.abs()) * w.double().abs() + 4 * U * h.abs()
            pad = -H % 128
            blocks = lambda t: torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (-1, 128))  # noqa: E731
            ref = blocks(h.abs()).amax(-1).clamp(min=1e-10) / 448.0
            assert scale.shape == ref.shape and q.shape == y.shape
            assert bool(((scale.double() - ref).abs() <= blocks(off).amax(-1) / 448.0 + 4 * U * ref).all())
            near_to = h / B.spread(scale, H, -1)
            step = torch.exp2(torch.floor(torch.log2(near_to.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0) - 3.0)
            got = q.double()
            assert bool(((got - near_to).abs() <= 0.5 * step * (1 + 2.0 ** -10) + off / B.spread(scale, H, -1) + 1e-9 + 4 * U * near_to.abs()).all())


def test_rows_of_extremes(dev):
    from gridbook_b200 import kernels
    for H in (64, 61):
        y = torch.zeros(4, H, device=dev)
        r = torch.zeros(4, H, device=dev)
        y[1, 3], r[2, 5] = float("nan"), float("inf")
        y[3] = 1e-30
        w = torch.ones(H, device=dev)
        h, s = kernels.residual_norm(y, r, w, post_weight=w, eps=1e-6)
        assert not bool(h[0].any()) and not bool(s[0].any())                 # a row of zeros stays one
        assert bool(torch.isnan(h[1]).all()) and bool(torch.isnan(s[1]).all())
        assert float(s[2, 5]) == float("inf") and bool(torch.isnan(h[2, 5])) and not bool(h[2, :5].any())
        assert bool(torch.isfinite(h[3]).all())
        assert kernels.residual_norm(y[:0], r[:0], w)[0].shape == (0, H)
    a, w = torch.zeros(0, 32, device=dev, requires_grad=True), torch.ones(32, device=dev, requires_grad=True)
    h, s = kernels.residual_norm(a, a, w)
    da, dw = torch.autograd.grad([h, s], [a, w], [torch.zeros_like(h), torch.zeros_like(s)])
    assert da.shape == a.shape and not bool(dw.any())


def test_strides_and_refusals(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 8)
    base = torch.randn(3, 40, 300, generator=g, device=dev).to(BF)
    w = torch.randn(256, generator=g, device=dev).to(BF)
    for cut in (lambda t: t[:, 8:264], lambda t: t[:, 3:259], lambda t: t[::2, :256], lambda t: t.t()[:256].t()):
        y, r, gt = (cut(t) for t in base)
        for leaf in (y, r, gt):
            assert not leaf.is_contiguous()
        got = kernels.residual_norm(y, r, w, post_weight=w, gate=gt, residual_scale=A, branch_scale=BR, eps=EPS)
        # rows that are no 16-byte pieces are added up in another order than contiguous ones: held to the formula, not to their bits
        want, size = stream_of(y, r, w, gt)
        near(got[1], want, (er(256) + 8 * U) * size, "stream")
        ref = rms(got[1].double()) * w.double()
        near(got[0], ref, (er(256) + 8 * U) * ref.abs(), "h")
        wide = torch.stack([w, w], 1)[:, 0]                                 # weights two apart
        assert torch.equal(kernels.residual_norm(y, r, wide, post_weight=w, gate=gt, residual_scale=A, branch_scale=BR, eps=EPS)[0], got[0])
    # gradients that are broadcast numbers or lie elsewhere than on 16-byte pieces
    y = torch.randn(8, 256, generator=g, device=dev).to(BF).requires_grad_()
    h, s = kernels.residual_norm(y, base[0, :8, :256], w, post_weight=w)
    one, ds = torch.ones((), device=dev, dtype=BF).expand(8, 256), base[1, :8, 3:259]
    d1, = torch.autograd.grad([h, s], [y], [one, ds])
    near(d1, *grads(s.detach(), y.detach(), w, w, None, one, ds, scales=(1.0, 1.0), eps=1e-6)["y"], "y")
    y, r = base[0, :, :256], base[1, :, :256]
    for call, kind in ((lambda: kernels.residual_norm(y, r[:4], w), RuntimeError), (lambda: kernels.residual_norm(y, r.half(), w), RuntimeError),
                       (lambda: kernels.residual_norm(y.double(), r.double()), TypeError), (lambda: kernels.residual_norm(y, r, w[:9]), RuntimeError),
                       (lambda: kernels.residual_norm(y, r, w.int()), TypeError), (lambda: kernels.residual_norm(y, r, w.cpu()), RuntimeError),
                       (lambda: kernels.residual_norm(y, r, gate=w.float()), RuntimeError), (lambda: kernels.residual_norm(y, r, gate=w[:9]), RuntimeError),
                       (lambda: kernels.residual_norm(y, r, gate=base[0, :39, :256]), RuntimeError),
                       (lambda: kernels.residual_norm(y.reshape(5, 8, 256), r.reshape(5, 8, 256), gate=y[:8]), RuntimeError),
                       (lambda: kernels.residual_norm_fp8(y.clone().requires_grad_(), r), RuntimeError)):
        with pytest.raises(kind):
            call()
    a = y.clone().requires_grad_()
    h, s = kernels.residual_norm(a, r, w)
    with pytest.raises(RuntimeError, match="no derivatives of their own"):
        torch.autograd.grad(h.sum(), a, create_graph=True)
    h, s = kernels.residual_norm(a, r, w)
    with torch.no_grad():
        s.add_(1)                                          # the backward pass would read it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_gradients_against_differences(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 14)
    y, r, w, pw, gt = (t.double() for t in _inputs(3, 24, F32, F32, "full", True, g, dev))
    dh, ds = torch.randn(3, 24, generator=g, device=dev), torch.randn(3, 24, generator=g, device=dev)

    def f(*t):
        h, s = kernels.residual_norm(t[0], t[1], t[2], post_weight=t[3], gate=t[4], residual_scale=A, branch_scale=BR, eps=EPS)
        return (h * dh).sum() + (s * ds).sum()
    base = [t.float() for t in (y, r, w, pw, gt)]
    leaves = [t.clone().requires_grad_() for t in base]
    got = torch.autograd.grad(f(*leaves), leaves)
    step = 2.0 ** -6
    for i, at in ((0, (1, 5)), (1, (2, 0)), (2, (7,)), (3, (23,)), (4, (0, 11))):
        up, down = [t.clone() for t in base], [t.clone() for t in base]
        up[i][at] += step
        down[i][at] -= step
        # third derivatives of order ten times step^2 / 6; roundings of sums of some 150 terms of order one over the step
        assert abs(float((f(*up) - f(*down)) / (2 * step)) - float(got[i][at])) < 10 * step ** 2 + 150 * U * 8 / step


def test_streams_graphs_and_many_rows(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 15)
    H = 512
    sets = [_inputs(700, H, BF, BF, "channel", True, g, dev) for _ in range(3)]
    dh, ds = (torch.randn(700, H, generator=g, device=dev).to(BF) for _ in range(2))

    def step(t):
        h, s = kernels.residual_norm(t[0], t[1], t[2], post_weight=t[3], gate=t[4], residual_scale=A)
        return (h.detach(), s.detach(), *torch.autograd.grad([h, s], list(t), [dh, ds]))
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
            for a, b in zip(t, sets[k]):
                a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, eager[k]))


def test_past_two_to_the_31_values(dev):
    from gridbook_b200 import kernels
    T, H = 300000, 7168                                     # 2.15e9 values, 4.3 GB a matrix
    y = torch.zeros(T, H, dtype=BF, device=dev)
    r = torch.zeros(T, H, dtype=BF, device=dev)
    g = _gen(dev, 16)
    y[-3:], r[-3:] = torch.randn(3, H, generator=g, device=dev).to(BF), torch.randn(3, H, generator=g, device=dev).to(BF)
    w = torch.randn(H, generator=g, device=dev).to(BF)
    h, s = kernels.residual_norm(y, r, w, post_weight=w)
    h2, s2 = kernels.residual_norm(y[-3:], r[-3:], w, post_weight=w)
    assert torch.equal(h[-3:], h2) and torch.equal(s[-3:], s2) and not bool(s[-100:-3].any())
    q, scale, _ = kernels.residual_norm_fp8(y, r, w, post_weight=w)
    q2, scale2, _ = kernels.residual_norm_fp8(y[-3:], r[-3:], w, post_weight=w)
    assert torch.equal(q[-3:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale[-3:], scale2)
