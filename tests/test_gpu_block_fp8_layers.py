"""The block-scaled layers as a user has them: the linear and the routed layer through their modules, their operators, under capture,
and a run of the operators one by one against the routed layer's single call."""
import pytest
import torch

from tests import blocks as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _experts(E, H, I, g, dev):
    return (*B.weights((E, 2 * I, H), g, dev), *B.weights((E, H, I), g, dev))


def _routing(T, E, topk, g, dev, extra=0):
    w, ids = torch.softmax(torch.randn(T, E + extra, generator=g, device=dev), -1).topk(topk, -1)
    return w / w.sum(-1, keepdim=True), ids


@pytest.mark.parametrize("M", [1, 5, 200])
def test_linear_module(dev, M):
    from gridbook_b200.block_fp8 import BlockFP8Linear
    g = _gen(dev, M)
    w, s = B.weights((520, 1040), g, dev)
    lin = BlockFP8Linear(1040, 520).load(w.cpu(), s.cpu(), dev)
    x = torch.randn(M, 1040, generator=g, device=dev).to(torch.bfloat16)
    y = lin(x)
    q, qs = B.quantize(x)
    B.assert_product(y, B.dequant_rows(q.to(dev), qs.to(dev)), B.dequant_weight(w, s), "module")
    assert torch.equal(torch.ops.prismaquant.fp8_blocks_linear(x, lin.weight, lin.weight_scale), y)
    assert torch.equal(lin(x.clone().requires_grad_()).detach(), y)        # through the operator
    state = lin.state_dict()
    assert set(state) == {"weight", "weight_scale"} and state["weight"].dtype is torch.float8_e4m3fn


CASES = [(1, 8, 2, 256, 128, 0), (3, 4, 4, 400, 272, 3), (40, 16, 4, 512, 384, 0), (700, 8, 2, 640, 256, 4), (16, 128, 8, 2048, 768, 0), (333, 2, 1, 128, 16, 0)]


@pytest.mark.parametrize("T,E,topk,H,I,extra", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_routed_layer(dev, dtype, T, E, topk, H, I, extra):
    """Bit for bit what the operators give one after the other, and the chain in 64 bits.  Between the projections a value next to a
    rounding boundary may land on the other side: one E4M3 step, 2^-3 of it (or 2^-9 scales among the subnormals), and the half
    step 2^-4 both round by; the first projection's and the rows' own rounding and sums are far below 2^-5 of the magnitudes
    that meet in them.  So the bound is that share of the sum of magnitudes of the second projection."""
    from gridbook_b200 import kernels
    from gridbook_b200.block_fp8 import BlockFP8MoE
    g = _gen(dev, T * E + H)
    w13, s13, w2, s2 = _experts(E, H, I, g, dev)
    moe = BlockFP8MoE(E, H, I, expert_base=extra // 2).load(w13, s13, w2, s2, dev)
    x = torch.randn(T, H, generator=g, device=dev).to(dtype)
    weights, ids = _routing(T, E, topk, g, dev, extra)
    out = moe(x, weights, ids)
    r = kernels.moe_sort(ids, E, expert_base=extra // 2)
    q, qs = kernels.moe_permute_fp8(x, r)
    h = kernels.gemm_fp8_blocks_grouped(q, qs, w13, s13, r.offsets, out_dtype=dtype)
    v, vs = kernels.moe_swiglu_fp8(h, r.offsets)
    y = kernels.gemm_fp8_blocks_grouped(v, vs, w2, s2, r.offsets, out_dtype=dtype)
    steps = kernels.moe_unpermute(y, r, weights)
    assert out.dtype is dtype and torch.equal(out, steps)
    assert torch.equal(torch.ops.prismaquant.fp8_blocks_moe(x, w13, s13, w2, s2, weights, ids.int(), extra // 2), out)
    rq, rs = B.quantize(x)
    a = B.dequant_rows(rq.to(dev), rs.to(dev))
    ref, size = torch.zeros(T, H, dtype=torch.float64, device=dev), torch.zeros(T, H, dtype=torch.float64, device=dev)
    for t in range(T):
        for k in range(topk):
            e = int(ids[t, k]) - extra // 2
            if not 0 <= e < E:
                continue
            gate, up = (a[t] @ B.dequant_weight(w13[e], s13[e]).T).chunk(2)
            act = gate / (1 + torch.exp(-gate)) * up
            block = torch.nn.functional.pad(act, (0, -I % 128)).view(-1, 128).abs().amax(-1).clamp(min=1e-10) / 448
            spread = block.repeat_interleave(128)[:I]
            val = B.e4m3_round(act / spread) * spread
            down = B.dequant_weight(w2[e], s2[e])
            ref[t] += float(weights[t, k]) * (down @ val)
            # what a value may be off by, the magnitudes that its gate and up are sums of included
            near = (2.0 ** -3 + 2.0 ** -4) * val.abs() + 2.0 ** -9 * spread
            in_size = (a[t].abs() @ B.dequant_weight(w13[e], s13[e]).abs().T).chunk(2)
            near += 2.0 ** -7 * (in_size[0] * up.abs() + in_size[1] * gate.abs()) * 2.0 ** -7 + 2.0 ** -7 * act.abs()
            size[t] += float(weights[t, k]) * (down.abs() @ near)
        if t >= 40:
            break
    n = min(T, 41)
    half = B.HALF[dtype]
    assert bool(((out[:n].double() - ref[:n]).abs() <= size[:n] + 4 * half * ref[:n].abs() + 1e-30).all())
    rel = float((out[:n].double() - ref[:n]).norm() / ref[:n].norm().clamp(min=1e-30))
    assert rel <= 2.0 ** -4 or float(ref[:n].norm()) == 0.0                # a step of E4M3 everywhere would be twice that


def test_routed_layer_shapes_and_nothing(dev):
    from gridbook_b200.block_fp8 import BlockFP8MoE
    g = _gen(dev, 3)
    moe = BlockFP8MoE(4, 256, 128).load(*_experts(4, 256, 128, g, dev), dev)
    x = torch.randn(6, 300, generator=g, device=dev).to(torch.bfloat16)
    w, ids = _routing(6, 4, 2, g, dev)
    whole = moe(x[:, 8:264].contiguous(), w, ids)
    assert torch.equal(moe(x[:, 8:264], w, ids), whole)
    assert torch.equal(moe(x[:, 8:264].reshape(2, 3, 256), w, ids), whole.view(2, 3, 256))
    assert torch.equal(moe(x[:, 8:264], w.to(torch.bfloat16).float().to(torch.bfloat16), ids), moe(x[:, 8:264], w.to(torch.bfloat16), ids.int()))
    assert moe(x[:0, :256], w[:0], ids[:0]).shape == (0, 256)
    none = moe(x[:, :256], w, torch.full_like(ids, -1))                    # every route is padding
    assert not bool(none.any())
    assert torch.equal(moe(x[:, 8:264], w, torch.stack([ids[:, 0], ids[:, 0]], 1)), moe(x[:, 8:264], w, torch.stack([ids[:, 0], ids[:, 0]], 1)))


def test_layers_in_a_graph_replayed_on_new_values(dev):
    from gridbook_b200.block_fp8 import BlockFP8Linear, BlockFP8MoE
    g = _gen(dev, 8)
    lin = BlockFP8Linear(512, 640).load(*B.weights((640, 512), g, dev), dev)
    moe = BlockFP8MoE(16, 640, 256).load(*_experts(16, 640, 256, g, dev), dev)
    for T in (1, 8, 300):
        xs = [torch.randn(T, 512, generator=g, device=dev).to(torch.bfloat16) for _ in range(3)]
        routes = [_routing(T, 16, 4, g, dev) for _ in range(3)]
        eager = [moe(lin(x), *r) for x, r in zip(xs, routes)]
        x, w, ids = xs[0].clone(), routes[0][0].clone(), routes[0][1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = moe(lin(x), w, ids)
        for i in (1, 2, 0):
            x.copy_(xs[i])
            w.copy_(routes[i][0])
            ids.copy_(routes[i][1])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[i])


def test_two_streams_at_once(dev):
    """The same layers called on two streams without a wait between the calls: nothing of a call is shared."""
    from gridbook_b200.block_fp8 import BlockFP8Linear, BlockFP8MoE
    g = _gen(dev, 9)
    lin = BlockFP8Linear(2048, 640).load(*B.weights((640, 2048), g, dev), dev)
    moe = BlockFP8MoE(16, 640, 256).load(*_experts(16, 640, 256, g, dev), dev)
    xs = [torch.randn(24, 2048, generator=g, device=dev).to(torch.bfloat16) for _ in range(2)]
    routes = [_routing(24, 16, 4, g, dev) for _ in range(2)]
    want = [moe(lin(x), *r) for x, r in zip(xs, routes)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(moe(lin(xs[i]), *routes[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_refusals(dev):
    from gridbook_b200.block_fp8 import BlockFP8Linear, BlockFP8MoE
    g = _gen(dev, 4)
    w, s = B.weights((128, 256), g, dev)
    lin = BlockFP8Linear(256, 128).load(w, s, dev)
    with pytest.raises(RuntimeError):
        lin(torch.zeros(2, 128, device=dev))
    with pytest.raises(RuntimeError):
        lin(torch.zeros(2, 256))
    moe = BlockFP8MoE(4, 256, 128).load(*_experts(4, 256, 128, g, dev), dev)
    x, (tw, ids) = torch.zeros(3, 256, device=dev), _routing(3, 4, 2, g, dev)
    for args in ((x[:2], tw, ids), (x[:, :128], tw, ids), (x, tw[:2], ids), (x, tw, ids[0]), (x, tw, ids.float()), (x, tw.cpu(), ids)):
        with pytest.raises(RuntimeError):
            moe(*args)
