"""What the router, the residual norms and the 16-bit linears refuse, told on the host: no GPU needed."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture(scope="module")
def lib():
    from gridbook_b200 import _native
    return _native.load()


def _text(lib):
    return lib.gb_last_error().decode()


P = ctypes.c_void_p(4096)          # an aligned address that no call below gets as far as reading
ODD = ctypes.c_void_p(4097)
NULL = ctypes.c_void_p(0)


@pytest.mark.parametrize("args,word", [
    ((P, 3, 8, 4, 8, 2, 0, 1, 1.0, P, P, NULL), "type"),
    ((P, 0, 8, 4, 0, 2, 0, 1, 1.0, P, P, NULL), "experts"),
    ((P, 0, 5000, 4, 4097, 2, 0, 1, 1.0, P, P, NULL), "experts"),
    ((P, 0, 8, 1 << 31, 8, 2, 0, 1, 1.0, P, P, NULL), "tokens"),
    ((P, 0, 7, 4, 8, 2, 0, 1, 1.0, P, P, NULL), "overlap"),
    ((ODD, 0, 8, 4, 8, 2, 0, 1, 1.0, P, P, NULL), "whole elements"),
    ((P, 0, 8, 4, 8, 0, 0, 1, 1.0, P, P, NULL), "top-0"),
    ((P, 0, 8, 4, 8, 9, 0, 1, 1.0, P, P, NULL), "top-9"),
    ((P, 0, 64, 4, 64, 33, 0, 1, 1.0, P, P, NULL), "top-33"),
    ((P, 0, 8, 4, 8, 2, 0, 1, 1.0, NULL, P, NULL), "null"),
])
def test_choice_refuses(lib, args, word):
    assert lib.gb_moe_topk(*args) != 0 and word in _text(lib)


def test_balance_refuses(lib):
    def call(logits=P, dtype=0, ld=8, ids=P, id_bytes=4, T=4, E=8, topk=2, loss=P):
        return lib.gb_moe_balance(logits, dtype, ld, ids, id_bytes, NULL, T, E, topk, 0.1, 0.0, loss, P, P, P, 1 << 20, NULL)
    for kw, word in ((dict(dtype=7), "type"), (dict(E=0), "experts"), (dict(id_bytes=2), "bytes"), (dict(topk=0), "one choice"), (dict(T=0), "one token"),
                     (dict(T=1 << 30), "pairs"), (dict(ids=NULL), "null"), (dict(ld=4), "overlap"), (dict(loss=NULL), "null")):
        assert call(**kw) != 0 and word in _text(lib), kw
    assert lib.gb_moe_balance_grad(P, 0, 8, NULL, NULL, P, 4, 8, 0.1, 0.0, P, NULL) != 0 and "null" in _text(lib)


def _norm(**kw):
    from gridbook_b200 import _native as nat
    args = dict(T=4, H=64, y=4096, r=4096, y_ld=64, r_ld=64, gate_ld=64, gate_rows=4, residual_scale=1.0, branch_scale=1.0, eps=1e-6)
    return nat.GbResidualNorm(**(args | kw))


def test_norms_refuse(lib):
    from gridbook_b200 import _native as nat
    for kw, word in ((dict(dtype=5), "type"), (dict(dtype=2, stream_dtype=0), "stream"), (dict(dtype=0, stream_dtype=1), "stream"), (dict(H=0), "shape"),
                     (dict(T=1 << 31), "shape"), (dict(w=4096, w_dtype=9), "weight type"), (dict(gate=4096, gate_rows=3), "gate rows"), (dict(y_ld=63), "overlap"),
                     (dict(gate=4096, gate_ld=8), "overlap"), (dict(y=None), "null")):
        a = _norm(**kw)
        assert lib.gb_residual_norm(ctypes.byref(a), P, P, NULL, NULL, NULL) != 0 and word in _text(lib), kw
    a = _norm()
    assert lib.gb_residual_norm_fp8(ctypes.byref(a), 5, P, P, P, NULL) != 0 and "rule" in _text(lib)
    g = nat.GbResidualNormGrads(stream=4096, rstd=4096, d_w=4096)
    assert lib.gb_residual_norm_grad(ctypes.byref(a), ctypes.byref(g), P, 1 << 30, NULL) != 0 and "there is not" in _text(lib)
    g = nat.GbResidualNormGrads(stream=4096)
    assert lib.gb_residual_norm_grad(ctypes.byref(a), ctypes.byref(g), P, 1 << 30, NULL) != 0 and "null" in _text(lib)


@pytest.mark.parametrize("args,word", [
    ((P, 64, P, NULL, NULL, 0, 2, 4, 8, 64, 0, P, NULL, NULL), "bf16 or fp16"),
    ((P, 64, P, NULL, NULL, 0, 0, 0, 8, 64, 0, P, NULL, NULL), "shape"),
    ((P, 64, P, NULL, NULL, 0, 0, 4, 1 << 31, 64, 0, P, NULL, NULL), "shape"),
    ((P, 64, P, NULL, NULL, 0, 0, 4, 8, 60, 0, P, NULL, NULL), "multiple of 8"),
    ((P, 64, NULL, NULL, NULL, 0, 0, 4, 8, 64, 0, P, NULL, NULL), "null"),
    ((P, 64, P, NULL, NULL, 0, 0, 4, 8, 64, 5, P, NULL, NULL), "activation"),
    ((P, 60, P, NULL, NULL, 0, 0, 4, 8, 56, 0, P, NULL, NULL), "16-byte"),
    ((ODD, 64, P, NULL, NULL, 0, 0, 4, 8, 64, 0, P, NULL, NULL), "16-byte"),
    ((P, 64, P, NULL, P, 7, 0, 4, 8, 64, 0, P, NULL, NULL), "overlap"),
])
def test_linear_refuses(lib, args, word):
    assert lib.gb_linear_act(*args) != 0 and word in _text(lib)


def test_linear_gradients_refuse(lib):
    def call(dy=P, dy_ld=8, z=P, x=P, x_ld=64, w=P, act=1, dx=P, dw=P, K=64):
        return lib.gb_linear_act_grad(dy, dy_ld, z, x, x_ld, w, 0, 4, 8, K, act, dx, dw, P, P, 1 << 30, NULL)
    for kw, word in ((dict(z=NULL), "null"), (dict(x=NULL), "null"), (dict(w=NULL), "null"), (dict(act=8), "activation"), (dict(dy_ld=7), "overlap"),
                     (dict(x_ld=60), "overlap"), (dict(K=4), "multiple of 8"), (dict(dw=ODD), "16-byte")):
        assert call(**kw) != 0 and word in _text(lib), kw


def test_empty_calls_launch_nothing(lib):
    before = lib.gb_launch_count()
    assert lib.gb_moe_topk(NULL, 0, 8, 0, 8, 2, 0, 1, 1.0, NULL, NULL, NULL) == 0
    assert lib.gb_moe_topk_grad(NULL, 0, 8, NULL, NULL, 0, 8, 2, 0, 1, 1.0, NULL, NULL) == 0
    a = _norm(T=0, y=None, r=None)
    assert lib.gb_residual_norm(ctypes.byref(a), NULL, NULL, NULL, NULL, NULL) == 0
    assert lib.gb_launch_count() == before


def test_host_tensors_and_unknown_words_are_refused():
    from gridbook_b200 import kernels
    x, l, ids = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: kernels.moe_topk(l, 2), lambda: kernels.moe_balance_loss(l, ids), lambda: kernels.residual_norm(x, x),
                 lambda: kernels.residual_norm_fp8(x, x), lambda: kernels.linear_act(x, x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(ValueError, match="tanh"):
        kernels.linear_act(x, x, activation="tanh")


def test_tangents_are_refused():
    from gridbook_b200 import kernels
    x, l, ids = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32)
    with fwd.dual_level():
        dx, dl = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(l, torch.ones_like(l))
        for call in (lambda: kernels.residual_norm(dx, x), lambda: kernels.residual_norm(x, dx), lambda: kernels.residual_norm_fp8(x, x, gate=dx),
                     lambda: kernels.linear_act(x, dx), lambda: kernels.linear_act(x, x, residual=dx)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
