"""16-bit linears whose sums pass fp16: the kept argument of the activation is infinite, its slope is not."""
import math

import pytest
import torch

from tests.blocks import HALF

pytestmark = pytest.mark.gpu
HF = torch.float16
F = torch.nn.functional
FN = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}
ADD, H, LOW = 2.0 ** -23, HALF[HF], 2.0 ** -25


def _close(got, ref, err, name):
    """Half a step of fp16 and ``err``; what rounds past its largest value is infinite."""
    past = ref.abs() >= 65520.0
    assert torch.equal(got[past].double(), torch.copysign(torch.full_like(ref[past], math.inf), ref[past])), name
    got, ref, err = got[~past], ref[~past], err[~past]
    off = (got.double() - ref).abs() - (err + (1 + 2.0 ** -8) * H * ref.abs() + LOW)
    assert bool(torch.isfinite(got).all()) and float(off.max()) <= 0.0, (name, float(off.max()))


@pytest.mark.parametrize("act", list(FN))
@pytest.mark.parametrize("M,N,K", [(3, 40, 256), (3, 4096, 1024), (60, 520, 256), (61, 523, 256), (700, 2304, 256), (701, 2305, 256)])
def test_sums_past_the_largest_value(act, M, N, K):
    """One row meets two weights whose products sum up to -131072 and 131072, and a bias does the rest for another."""
    from gridbook_b200 import kernels
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(M + N)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)
    x, w, b = normal(M, K), normal(N, K) * (1.5 / math.sqrt(K)), normal(N)
    x[0] = 64.0
    w[3], w[5], w[7] = -2048.0 / K, 2048.0 / K, -1000.0 / K
    b[7] = -30000.0
    x, w, b = (t.to(HF).requires_grad_() for t in (x, w, b))
    dy = normal(M, N).to(HF)
    y = kernels.linear_act(x, w, b, activation=act)
    got = torch.autograd.grad(y, [x, w, b], dy)
    xd, wd, bd = (t.detach().double() for t in (x, w, b))
    z, size = xd @ wd.T + bd, xd.abs() @ wd.abs().T + bd.abs()
    assert float(z[0, 3]) < -65520 and float(z[0, 5]) > 65520 and float(z[0, 7]) < -65520
    ez = (K + 2) * ADD * size
    # (the activations' steepest slope 1.13, a few units of the argument for the function itself)
    _close(y.detach(), FN[act](z), torch.where(z < -60.0, 0.0 if act else 1.0, 1.0) * 1.13 * ez + 16 * ADD * z.abs().clamp(max=60.0 if act else math.inf), f"y {act}")
    zl = z.clone().requires_grad_()
    slope, = torch.autograd.grad(FN[act](zl).sum(), zl)
    dz, d = dy.double() * slope, dy.double().abs()
    ek = ez + H * z.abs() + LOW                               # of z as it is kept; past 60 the slopes are constant to more than fp32's digits
    flat = z.abs() > 60.0 + ek
    if act is None:
        e = torch.zeros_like(z)
    elif act == "relu":
        e = d * (z.abs() <= ek)
    else:
        e = d * (torch.where(flat, 0.0, 0.8 * ek) + 2.0 ** -20)
    db_err = e.sum(0) + (M + 4) * 2.0 ** -24 * dz.abs().sum(0)
    if act:
        e = e + H * (dz.abs() + e) + LOW
    s = dz.abs() + e
    _close(got[0], dz @ wd, e @ wd.abs() + (N + 2) * ADD * (s @ wd.abs()), f"dx {act}")
    _close(got[1], dz.T @ xd, e.T @ xd.abs() + (M + 18) * ADD * (s.T @ xd.abs()), f"dw {act}")
    _close(got[2], dz.sum(0), db_err, f"db {act}")
