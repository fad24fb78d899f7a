"""Plain 64-bit forms of the block-scaled E4M3 operators and of the tokens' sort, for the tests."""
import torch

BLOCK = 128
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}     # half a step, relative


def spread(scale, n, dim):
    """One scale per element along ``dim`` from one per block."""
    return scale.double().repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def dequant_rows(q, scale):
    return q.double() * spread(scale, q.shape[-1], -1)


def dequant_weight(w, scale):
    return w.double() * spread(spread(scale, w.shape[-2], -2), w.shape[-1], -1)


def e4m3_round(v):
    """The nearest E4M3 value of fp64 values, ties to even, saturating; NaN stays."""
    mag = v.abs().clamp(min=2.0 ** -30)
    step = torch.exp2(torch.floor(torch.log2(mag)).clamp(min=-6.0) - 3.0)
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def quantize(x, rule="recip"):
    """(E4M3 values as fp64, fp32 scale): the scale a product in fp32 with the reciprocal or a true division, the quotient
    rounded to fp32 and then to E4M3.  On the CPU, where torch divides by a number as it says."""
    x = x.detach().float().cpu()
    k = x.shape[-1]
    xb = torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = xb.abs().amax(-1)                                     # spreads a NaN
    amax = torch.where(amax < 1e-10, torch.full_like(amax, 1e-10), amax)
    top = torch.full_like(amax, 448.0)
    scale = amax / top if rule == "div" else amax * (torch.ones_like(amax) / top)
    q = e4m3_round((xb / scale.unsqueeze(-1)).double()).flatten(-2)[..., :k]
    return q, scale


def weights(shape, gen, dev):
    """Random E4M3 weights [.., N, K] and their scales."""
    *lead, n, k = shape
    w = (torch.randn(*shape, generator=gen, device=dev) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(*lead, -(-n // BLOCK), -(-k // BLOCK), generator=gen, device=dev) * 0.002 + 0.0005
    return w, s


def rows(m, k, gen, dev):
    a = (torch.randn(m, k, generator=gen, device=dev) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return a, torch.rand(m, -(-k // BLOCK), generator=gen, device=dev) * 0.02 + 0.002


def assert_product(got, a, b, tag):
    """``got`` against a . b^T of fp64 operands.  Error: half a step of the output's type, and fp32 adds: 128 terms of a block and
    the blocks, each add off by at most a whole unit (how the tensor cores round theirs is not specified), two products of
    scales."""
    ref, size = a @ b.T, a.abs() @ b.abs().T
    n = BLOCK + -(-a.shape[1] // BLOCK) + 4
    tol = HALF[got.dtype] * ref.abs() + (1 + HALF[got.dtype]) * n * 2.0 ** -23 * size + (2.0 ** -25 if got.dtype is torch.float16 else 0.0)
    off = (got.double() - ref).abs() - tol
    assert bool(torch.isfinite(got).all()), f"{tag}: not finite"
    assert float(off.max()) <= 0.0, f"{tag}: {int((off > 0).sum())} of {off.numel()} off, by up to {float(off.max()):.3e}"


def sort(ids, E, base=0):
    """counts, offsets, order, place of the pairs in expert order, as lists."""
    flat = [int(i) - base for i in ids.reshape(-1).tolist()]
    live = sorted((p for p in range(len(flat)) if 0 <= flat[p] < E), key=flat.__getitem__)
    counts = [0] * E
    for p in live:
        counts[flat[p]] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    place = [-1] * len(flat)
    for j, p in enumerate(live):
        place[p] = j
    return counts, offsets, live + [0] * (len(flat) - len(live)), place
