"""What the operators around the routed and linear layers are measured on: a 16-bit linear with bias, activation and residual in its
epilogue, the norms behind and in front of a block with its gate and residual scale, the router's top-k, and its balance loss with
the experts' counts.  From one decode row to long prefills and training batches, with the gradients of all four.

With ``own`` false the plain form runs: elementary torch operations in 32 bits, rounded once at the end (values that the operator
stores and reads again, the residual stream, as they are stored)."""
import math

import torch

own = False

BLOCK = 128                 # columns of an E4M3 block of activations
AMAX_FLOOR = 1e-10          # smallest largest-magnitude of a block: a block of zeros gets a scale that divides
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # one decode row through a biased linear
        dict(name="linear_m1", kind="linear", dtype="bf16", M=1, N=4096, K=4096, bias=True, act="silu", residual=False, train=False),
        # the ragged tail of a chunked prefill through the down projection, onto the residual stream
        dict(name="linear_m333_down", kind="linear", dtype="bf16", M=333, N=5120, K=17408, bias=True, act="none", residual=True, train=False),
        # a long prefill through the widest linear of a 5120-wide layer
        dict(name="linear_m8192_gate_up", kind="linear", dtype="bf16", M=8192, N=34816, K=5120, bias=True, act="gelu_tanh", residual=False, train=False),
        # a training step of a linear: activation in the epilogue, gradients of rows, weight, bias and residual
        dict(name="linear_train_t4096", kind="linear", dtype="bf16", M=4096, N=8192, K=5120, bias=True, act="gelu", residual=True, train=True),
        # one decode row between two blocks: the smallest call, launch and call overhead
        dict(name="norm_m1", kind="norm", out="rows", dtype="bf16", stream="bf16", M=1, H=5120, post=True, gate="none", train=False),
        # a prefill's rows on the way into block-scaled FP8 layers: the norm's output quantised where it is made
        dict(name="norm_fp8_m4096", kind="norm", out="fp8", dtype="bf16", stream="bf16", M=4096, H=7168, post=True, gate="channel", train=False),
        # a training batch, layer-scale gate, gradients of everything
        dict(name="norm_train_t8192", kind="norm", out="rows", dtype="bf16", stream="bf16", M=8192, H=5120, post=True, gate="channel", train=True),
        # three ragged sequences with a gate each and the stream held in 32 bits
        dict(name="norm_train_t777_fp32", kind="norm", out="rows", dtype="fp32", stream="fp32", M=777, H=2056, post=True, gate="sequence", train=True),
        # one token's experts
        dict(name="topk_t1", kind="topk", dtype="bf16", T=1, E=128, topk=8, score="softmax", renormalize=True, train=False),
        # a training batch of the large routed layer, logits in 32 bits
        dict(name="topk_train_t8192", kind="topk", dtype="fp32", T=8192, E=256, topk=8, score="sigmoid", renormalize=True, train=True),
        # a short padded batch
        dict(name="balance_t333", kind="balance", dtype="fp32", T=333, E=128, topk=8, masked=True),
        # a training batch of many sequences
        dict(name="balance_t65536", kind="balance", dtype="bf16", T=65536, E=256, topk=8, masked=False),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "norm", "topk", "balance"])
    if kind == "linear":
        train = rng.random() < 0.5
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16"]), M=_log(rng, 1, 4096), N=_log(rng, 256, 16384, rng.choice([1, 8, 64, 128])),
                    K=_log(rng, 256, 8192, rng.choice([8, 64, 128])), bias=rng.random() < 0.7, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                    residual=rng.random() < 0.5, train=train)
    if kind == "norm":
        out = rng.choice(["rows", "rows", "fp8"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return dict(kind=kind, out=out, dtype=dtype, stream=rng.choice([dtype, "fp32"]), M=_log(rng, 1, 16384), H=_log(rng, 64, 8192, rng.choice([1, 8, 64, 128])),
                    post=rng.random() < 0.7, gate=rng.choice(["none", "channel", "sequence", "full"]), train=out == "rows" and rng.random() < 0.6)
    E = _log(rng, 8, 512)
    topk = min(E, rng.choice([1, 2, 4, 6, 8]))
    if kind == "topk":
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), T=_log(rng, 1, 32768), E=E, topk=topk, score=rng.choice(["softmax", "sigmoid"]),
                    renormalize=rng.random() < 0.7, train=rng.random() < 0.6)
    return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), T=_log(rng, 1, 32768), E=E, topk=topk, masked=rng.random() < 0.5)


# ------------------------------------------------------------------------------------- inputs
def _activations(m, k, gen, dev):
    """Rows as a norm leaves them: N(0, 1) times a scale for each column, a few columns far larger."""
    cols = torch.exp(0.5 * torch.randn(k, generator=gen, device=dev))
    cols = torch.where(torch.rand(k, generator=gen, device=dev) < 0.01, cols * 20.0, cols)
    return torch.randn(m, k, generator=gen, device=dev) * cols


def _sequences(m):
    """Sequences of a batch of ``m`` rows that have a gate each."""
    return next(n for n in (3, 7, 2, 5, 1) if m % n == 0)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = dict(case, dt=dt)
    train = bool(case.get("train", True))
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x = _activations(M, K, gen, dev)
        w = normal(N, K).mul_(1.0 / (2.0 * math.sqrt(K)))
        s["x"], s["w"] = x.to(dt).requires_grad_(train), w.to(dt).requires_grad_(train)
        s["b"] = normal(N).mul_(0.5).to(dt).requires_grad_(train) if case["bias"] else None
        s["r"] = normal(M, N).to(dt).requires_grad_(train) if case["residual"] else None
        s["dy"] = normal(M, N).to(dt) if train else None
    elif kind == "norm":
        M, H, st = case["M"], case["H"], DTYPES[case["stream"]]
        s["y"], s["r"] = _activations(M, H, gen, dev).to(dt).requires_grad_(train), normal(M, H).mul_(4.0).to(st).requires_grad_(train)
        s["w"] = (1.0 + 0.2 * normal(H)).to(dt).requires_grad_(train)
        s["pw"] = (1.0 + 0.2 * normal(H)).to(dt).requires_grad_(train) if case["post"] else None
        shape = {"none": None, "channel": (H,), "sequence": (_sequences(M), 1, H), "full": (M, H)}[case["gate"]]
        s["g"] = None if shape is None else (0.5 * normal(*shape)).to(dt).requires_grad_(train)
        if case["gate"] == "sequence":
            n = shape[0]
            s["y"], s["r"] = (t.detach().view(n, M // n, H).requires_grad_(train) for t in (s["y"], s["r"]))
        s["d_h"] = torch.randn(s["y"].shape, generator=gen, device=dev).to(dt) if train else None
        s["d_r"] = torch.randn(s["y"].shape, generator=gen, device=dev).to(st) if train else None
    else:
        T, E, topk = case["T"], case["E"], case["topk"]
        s["l"] = (1.5 * normal(T, E)).to(dt).requires_grad_(train)
        if kind == "topk":
            s["dw"] = normal(T, topk)
        else:
            ids = torch.topk(s["l"].detach().float() + 0.3 * normal(T, E), topk, -1).indices
            s["ids"] = ids.to(torch.int32).contiguous()
            s["mask"] = (torch.rand(T, generator=gen, device=dev) < 0.8) if case["masked"] else None
            s["dl"] = torch.full((), 0.7, device=dev)
    return s


RESIDUAL_SCALE, BRANCH_SCALE, ROUTE_SCALE, BALANCE, Z = 0.9, 1.1, 2.5, 1e-2, 1e-3


# ------------------------------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    return torch.ones_like(z)


def _linear(s):
    dt, x, w = s["dt"], s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = [y.to(dt)]
    if s["train"]:
        dz = s["dy"].float() * _act_slope(z, s["act"])
        out += [(dz @ w).to(dt), (dz.T @ x).to(dt)]
        if s["b"] is not None:
            out.append(dz.sum(0).to(dt))
        if s["r"] is not None:
            out.append(s["dy"])
    return out


def _quantize(x):
    """(E4M3 values, fp32 scale of every block of 128 columns), x ~ values * scale."""
    k = x.shape[-1]
    xb = torch.nn.functional.pad(x, (0, -(-k // BLOCK) * BLOCK - k)).unflatten(-1, (-1, BLOCK))
    scale = xb.abs().amax(-1).clamp(min=AMAX_FLOOR) * (1.0 / 448.0)
    q = (xb / scale.unsqueeze(-1)).clamp(-448.0, 448.0).flatten(-2)[..., :k]
    return q.to(E4M3), scale


def _norm(s):
    dt, y, w = s["dt"], s["y"].float(), s["w"].float()
    gate = BRANCH_SCALE if s["g"] is None else s["g"].float() * BRANCH_SCALE
    u = y
    if s["pw"] is not None:
        r_post = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        y_hat, pw = y * r_post, s["pw"].float()
        u = y_hat * pw
    x = s["r"].float() * RESIDUAL_SCALE + gate * u
    stream = x.to(s["r"].dtype)
    if s["out"] == "rows":                          # the norm of the stream as it is stored, from which the gradients start too
        x = stream.float()
    r_pre = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    x_hat = x * r_pre
    if s["out"] == "fp8":
        return [*_quantize(x_hat * w), stream]
    out = [(x_hat * w).to(dt), stream]
    if s["train"]:
        dh = s["d_h"].float()
        dxh = dh * w
        dx = s["d_r"].float() + r_pre * (dxh - x_hat * (dxh * x_hat).mean(-1, keepdim=True))
        du = dx * gate
        rows = tuple(range(dx.dim() - 1))
        dy = du
        if s["pw"] is not None:
            dyh = du * pw
            dy = r_post * (dyh - y_hat * (dyh * y_hat).mean(-1, keepdim=True))
        out += [dy.to(dt), (dx * RESIDUAL_SCALE).to(s["r"].dtype), (dh * x_hat).sum(rows).to(dt)]
        if s["pw"] is not None:
            out.append((du * y_hat).sum(rows).to(dt))
        if s["g"] is not None:
            dg = dx * u * BRANCH_SCALE
            out.append({"channel": lambda: dg.sum(rows), "sequence": lambda: dg.sum(1, keepdim=True), "full": lambda: dg}[s["gate"]]().to(dt))
    return out


def _topk(s):
    l, k = s["l"].float(), s["topk"]
    ids = torch.argsort(l, dim=-1, descending=True, stable=True)[:, :k]      # ties to the lowest index
    if s["score"] == "softmax":
        p = torch.exp(l - l.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    c = p.gather(1, ids)
    total = c.sum(-1, keepdim=True) if s["renormalize"] else torch.ones_like(c[:, :1])
    w = c / total * ROUTE_SCALE
    out = [w, ids.int()]
    if s["train"]:
        dc = s["dw"] * ROUTE_SCALE / total
        if s["renormalize"]:
            dc = dc - (dc * c).sum(-1, keepdim=True) / total
        dp = torch.zeros_like(p).scatter_(1, ids, dc)
        dl = p * (dp - (dp * p).sum(-1, keepdim=True)) if s["score"] == "softmax" else dp * p * (1.0 - p)
        out.append(dl.to(s["dt"]))
    return out


def _balance(s):
    l, E, k = s["l"].float(), s["E"], s["topk"]
    live = torch.ones_like(l[:, :1]) if s["mask"] is None else s["mask"].float().unsqueeze(-1)
    n = live.sum()
    top = l.amax(-1, keepdim=True)
    e = torch.exp(l - top)
    total = e.sum(-1, keepdim=True)
    p, lse = e / total, top + torch.log(total)
    counts = torch.zeros(E, device=l.device).scatter_add_(0, s["ids"].reshape(-1).long(), live.expand(-1, k).reshape(-1))
    some = n.clamp(min=1.0)
    f = counts / (some * k)
    loss = BALANCE * E * (f * (p * live).sum(0) / some).sum() + Z * ((lse * live).square().sum() / some)
    dl = s["dl"] * live / some * p * (BALANCE * E * (f - (f * p).sum(-1, keepdim=True)) + 2.0 * Z * lse)
    return [loss, counts.int(), dl.to(s["dt"])]


@torch.no_grad()
def _plain(s):
    return {"linear": _linear, "norm": _norm, "topk": _topk, "balance": _balance}[s["kind"]](s)


def run(state):
    if not own:
        return _plain(state)
    from gridbook_b200 import kernels

    s, kind = state, state["kind"]
    if kind == "linear":
        y = kernels.linear_act(s["x"], s["w"], s["b"], activation=None if s["act"] == "none" else s["act"], residual=s["r"])
        if not s["train"]:
            return [y]
        return [y, *torch.autograd.grad([y], [t for t in (s["x"], s["w"], s["b"], s["r"]) if t is not None], [s["dy"]])]
    if kind == "norm":
        call = kernels.residual_norm_fp8 if s["out"] == "fp8" else kernels.residual_norm
        out = call(s["y"], s["r"], s["w"], post_weight=s["pw"], gate=s["g"], residual_scale=RESIDUAL_SCALE, branch_scale=BRANCH_SCALE, eps=EPS)
        if not s["train"]:
            return list(out)
        return [*out, *torch.autograd.grad(list(out), [t for t in (s["y"], s["r"], s["w"], s["pw"], s["g"]) if t is not None], [s["d_h"], s["d_r"]])]
    if kind == "topk":
        w, ids = kernels.moe_topk(s["l"], s["topk"], score=s["score"], renormalize=s["renormalize"], scale=ROUTE_SCALE)
        return [w, ids, *torch.autograd.grad([w], [s["l"]], [s["dw"]])] if s["train"] else [w, ids]
    loss, counts = kernels.moe_balance_loss(s["l"], s["ids"], coef=BALANCE, z_coef=Z, mask=s["mask"])
    return [loss, counts, *torch.autograd.grad([loss], [s["l"]], [s["dl"]])]


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = DTYPES[case["dtype"]].itemsize
    kind, train = case["kind"], bool(case.get("train", True))
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        tiles = M * K + N * K + M * N * (1 + case["residual"]) + N * case["bias"]
        if train:                                   # the output's gradient in; of rows, weight and bias out (the residual's is the output's)
            tiles += M * N + M * K + N * K + N * case["bias"]
        return {"bytes": size * tiles, "flops": 2.0 * M * N * K * (3 if train else 1)}
    if kind == "norm":
        M, H, st = case["M"], case["H"], DTYPES[case["stream"]].itemsize
        full = case["gate"] == "full"
        if case["out"] == "fp8":
            return {"bytes": M * (H * (size * (1 + full) + 2 * st + 1) + 4 * -(-H // BLOCK)), "flops": 10.0 * M * H}
        per = size * (2 + full) + 2 * st            # y, gate, stream in; rows and stream out
        if train:                                   # gradients of rows and stream in; of y, gate and stream out
            per += size * (2 + full) + 2 * st
        return {"bytes": M * H * per, "flops": (30.0 if train else 8.0) * M * H}
    T, E, topk = case["T"], case["E"], case["topk"]
    if kind == "topk":
        return {"bytes": T * (size * E * (2 if train else 1) + 8 * topk + (4 * topk if train else 0)), "flops": (8.0 if train else 4.0) * T * E}
    return {"bytes": T * (2 * size * E + 4 * topk) + 4 * E, "flops": 16.0 * T * E}


# ------------------------------------------------------------------------------------- the definition, in 64 bits
def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_()


def _grads(outs, d_outs, leaves):
    return list(torch.autograd.grad(outs, leaves, [d.double() for d in d_outs]))


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    F = torch.nn.functional
    if kind == "linear":
        fn = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}[s["act"]]
        if not s["train"]:
            with torch.no_grad():
                x, y = s["x"].double(), torch.empty(case["M"], case["N"], dtype=torch.double, device=s["x"].device)
                for n in range(0, case["N"], 4096):
                    at = slice(n, n + 4096)
                    z = F.linear(x, s["w"][at].double(), None if s["b"] is None else s["b"][at].double())
                    y[:, at] = fn(z) + (0.0 if s["r"] is None else s["r"][:, at].double())
            return [y]
        leaves = [_leaf(s[k]) for k in ("x", "w", "b", "r")]
        x, w, b, r = leaves
        y = fn(F.linear(x, w, b))
        y = y if r is None else y + r
        return [y.detach(), *_grads([y], [s["dy"]], [t for t in leaves if t is not None])]
    if kind == "norm":
        leaves = [_leaf(s[k]) for k in ("y", "r", "w", "pw", "g")]
        y, r, w, pw, g = leaves
        H = (case["H"],)
        u = y if pw is None else F.rms_norm(y, H, pw, EPS)
        x = RESIDUAL_SCALE * r + BRANCH_SCALE * (u if g is None else g * u)
        if s["out"] == "rows":
            x = x + (x.detach().to(s["r"].dtype).double() - x.detach())   # as the stream stores it
        h = F.rms_norm(x, H, w, EPS)
        if s["out"] == "fp8":
            k = case["H"]
            hb = F.pad(h.detach(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
            scale = torch.linalg.vector_norm(hb, float("inf"), dim=-1).clamp(min=AMAX_FLOOR) / 448.0
            v = hb / scale.unsqueeze(-1)
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0) - 3.0)
            return [(torch.round(v / step) * step).clamp(-448.0, 448.0).flatten(-2)[..., :k], scale, x.detach()]
        out = [h.detach(), x.detach()]
        return out + (_grads([h, x], [s["d_h"], s["d_r"]], [t for t in leaves if t is not None]) if s["train"] else [])
    l = _leaf(s["l"])
    if kind == "topk":
        p = torch.softmax(l, -1) if s["score"] == "softmax" else torch.sigmoid(l)
        c = p.gather(1, torch.sort(l.detach(), dim=-1, descending=True, stable=True).indices[:, :s["topk"]])
        w = ROUTE_SCALE * (c / c.sum(-1, keepdim=True) if s["renormalize"] else c)
        return [w.detach(), None] + (_grads([w], [s["dw"]], [l]) if s["train"] else [])
    rows, ids = (l, s["ids"]) if s["mask"] is None else (l[s["mask"]], s["ids"][s["mask"]])
    n = rows.shape[0]
    if n == 0:
        return [torch.zeros((), dtype=torch.double, device=l.device), None, torch.zeros_like(l.detach())]
    f = torch.bincount(ids.reshape(-1).long(), minlength=case["E"]).double() / (n * case["topk"])
    loss = BALANCE * case["E"] * (f * torch.softmax(rows, -1).mean(0)).sum() + Z * torch.logsumexp(rows, -1).square().mean()
    return [loss.detach(), None, *_grads([loss], [s["dl"]], [l])]
