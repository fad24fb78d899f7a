"""The router, the residual norms, the 16-bit linears and the sorted rows as a routed block uses them together: a training step against
the same block in fp64, and a served token's way through block-scaled layers."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
F = torch.nn.functional


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _weights(H, I, E, g, dev):
    def n(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * by).to(BF).requires_grad_()
    return dict(pre=(1 + 0.1 * torch.randn(H, generator=g, device=dev)).to(BF).requires_grad_(), post=(1 + 0.1 * torch.randn(H, generator=g, device=dev)).to(BF).requires_grad_(),
                gate=n(H, by=0.5), router=n(E, H, by=2.0 * H ** -0.5), up=n(E, I, H, by=H ** -0.5), up_b=n(E, I, by=0.1), down=n(E, H, I, by=2.0 * I ** -0.5), down_b=n(E, H, by=0.1))


def test_training_step(dev):
    from gridbook_b200 import kernels
    g = _gen(dev, 1)
    T, H, I, E, k = 400, 256, 320, 6, 2
    p = _weights(H, I, E, g, dev)
    x, r = (torch.randn(T, H, generator=g, device=dev).to(BF).requires_grad_() for _ in range(2))
    d_h, d_s = (torch.randn(T, H, generator=g, device=dev).to(BF) for _ in range(2))
    seen = {}

    def step():
        h, s = kernels.residual_norm(x, r, p["pre"])
        logits = kernels.linear_act(h, p["router"])
        w, ids = kernels.moe_topk(logits, k)
        loss, counts = kernels.moe_balance_loss(logits, ids, coef=1.0, z_coef=0.1)
        srt = kernels.moe_sort(ids, E)
        rows = kernels.moe_permute(h, srt)
        ends = srt.offsets.tolist()
        parts = [kernels.linear_act(kernels.linear_act(rows[a:b], p["up"][e], p["up_b"][e], activation="silu"), p["down"][e], p["down_b"][e])
                 for e, (a, b) in enumerate(zip(ends, ends[1:]))]
        out = kernels.moe_unpermute(torch.cat(parts), srt, w)
        h2, s2 = kernels.residual_norm(out, s, p["pre"], post_weight=p["post"], gate=p["gate"], residual_scale=0.9)
        seen.update(ids=ids, counts=counts, loss=loss)
        assert torch.equal(counts, srt.counts)
        return [h2, s2, loss]

    def reference():
        """The same in fp64, for the experts that were chosen."""
        q = {n: t.detach().double().requires_grad_() for n, t in p.items()}
        xd, rd = (t.detach().double().requires_grad_() for t in (x, r))
        s = xd + rd
        h = F.rms_norm(s, (H,), q["pre"], 1e-6)
        logits = h @ q["router"].T
        probs, ids = torch.softmax(logits, -1), seen["ids"].long()
        c = probs.gather(1, ids)
        w = c / c.sum(-1, keepdim=True)
        f = torch.bincount(ids.reshape(-1), minlength=E).double() / (T * k)
        loss = E * (f * probs.mean(0)).sum() + 0.1 * torch.logsumexp(logits, -1).square().mean()
        every = torch.stack([F.silu(h @ q["up"][e].T + q["up_b"][e]) @ q["down"][e].T + q["down_b"][e] for e in range(E)], 1)
        out = (every.gather(1, ids[..., None].expand(-1, -1, H)) * w[..., None]).sum(1)
        s2 = 0.9 * s + q["gate"] * F.rms_norm(out, (H,), q["post"], 1e-6)
        h2 = F.rms_norm(s2, (H,), q["pre"], 1e-6)
        return [h2, s2, loss], [xd, rd, *q.values()]

    outs = step()
    grads = torch.autograd.grad(outs, [x, r, *p.values()], [d_h, d_s, torch.ones_like(outs[2])])
    ref, leaves = reference()
    want = torch.autograd.grad(ref, leaves, [d_h.double(), d_s.double(), torch.ones_like(ref[2])])
    # Some twenty roundings to bf16 lie on the longest way there and back, each off by 2^-8 / sqrt(3) in the mean, on maps that stretch
    # errors about as much as values: sqrt(20) 2^-8 / sqrt(3) = 1% of the norm, four times that is allowed.  The loss reads logits
    # rounded once.
    for name, a, b in zip(["h", "stream", "loss", "x", "r", *p], [*outs, *grads], [*ref, *want]):
        assert float((a.detach().double() - b.detach()).norm()) <= 0.04 * float(b.detach().norm()), name


def test_a_block_of_tokens_on_the_way_into_block_scaled_layers(dev):
    """The norm's E4M3 rows multiplied as they are; the router's choice in front of routed block-scaled experts, tokens that choose nobody
    among them."""
    from gridbook_b200 import kernels
    from gridbook_b200.block_fp8 import BlockFP8MoE
    g = _gen(dev, 2)
    H, I, E, k = 512, 256, 16, 4
    dense, dense_s = B.weights((384, H), g, dev)
    w13, s13 = B.weights((E, 2 * I, H), g, dev)
    w2, s2 = B.weights((E, H, I), g, dev)
    moe = BlockFP8MoE(E, H, I).load(w13, s13, w2, s2)
    norm = (1 + 0.1 * torch.randn(H, generator=g, device=dev)).to(BF)
    router = (torch.randn(E, H, generator=g, device=dev) * H ** -0.5).to(BF)
    for T in (1, 5, 130):
        y, r = (torch.randn(T, H, generator=g, device=dev).to(BF) for _ in range(2))
        q, scale, s = kernels.residual_norm_fp8(y, r, norm, post_weight=norm)
        B.assert_product(kernels.gemm_fp8_blocks(q, scale, dense, dense_s), B.dequant_rows(q, scale), B.dequant_weight(dense, dense_s), f"T={T}")
        h, s_again = kernels.residual_norm(y, r, norm, post_weight=norm)
        assert torch.equal(s, s_again)
        logits = kernels.linear_act(h, router)
        logits[T // 2] = float("-inf")
        w, ids = kernels.moe_topk(logits, k)
        out = moe(h, w, ids)
        assert not bool(out[T // 2].any()) and ids[T // 2].tolist() == [-1] * k
        keep = [t for t in range(T) if t != T // 2]
        if keep:
            assert torch.equal(out[keep], moe(h[keep], w[keep], ids[keep])) or float((out[keep].double() - moe(h[keep], w[keep], ids[keep]).double()).norm()) <= \
                B.HALF[BF] * 4 * float(out[keep].double().norm())      # other numbers of rows may take other tiles: sums in another order, one rounding apart


def test_a_captured_training_step_beside_eager_ones(dev):
    """Forward and backward of all four in one graph, replayed between eager steps on other leaves."""
    from gridbook_b200 import kernels
    g = _gen(dev, 3)
    T, H, E, k = 96, 256, 8, 2
    w, norm = (torch.randn(E, H, generator=g, device=dev) * H ** -0.5).to(BF), torch.ones(H, dtype=BF, device=dev)
    sets = [[torch.randn(T, H, generator=g, device=dev).to(BF) for _ in range(2)] for _ in range(3)]
    d = torch.randn(T, H, generator=g, device=dev).to(BF)

    def step(x, r, w, n):
        h, s = kernels.residual_norm(x, r, n, post_weight=n)
        logits = kernels.linear_act(h, w)
        c, ids = kernels.moe_topk(logits, k)
        loss, _ = kernels.moe_balance_loss(logits, ids, coef=1.0)
        srt = kernels.moe_sort(ids, E)
        out = kernels.moe_unpermute(kernels.moe_permute(h, srt), srt, c)
        return (out.detach(), loss.detach(), *torch.autograd.grad([out, s, loss], [x, r, w, n], [d, d, torch.ones_like(loss)]))

    def eager(i):
        return [t.clone() for t in step(*(t.clone().requires_grad_() for t in (*sets[i], w, norm)))]
    want = [eager(i) for i in range(3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        leaves = [t.clone().requires_grad_() for t in (*sets[0], w, norm)]
        step(*leaves)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(*leaves)
    for i in (1, 0, 2):
        with torch.no_grad():
            for a, b in zip(leaves, sets[i]):
                a.copy_(b)
        graph.replay()
        again = eager(i)
        torch.cuda.synchronize()
        for p, q, s in zip(res, want[i], again):
            assert torch.equal(p, q) and torch.equal(s, q)
