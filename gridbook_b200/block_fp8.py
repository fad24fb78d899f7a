"""Layers kept at a checkpoint's own block-scaled FP8: E4M3 weights with one fp32 scale per 128 x 128 block, activations quantised
per call in blocks of 128 columns.  They stand beside the codebook layers (:class:`~gridbook_b200.linear.CBLinear`,
:class:`~gridbook_b200.moe.CBMoE`) for the parts of a mixed-precision artifact that are not codebook-coded.  The reference
serves such layers outside its codebook path, multiplying bf16 activations (gridbook/fp8_source_w8a16.py).

Inference only, sm_100a only: a missing library or kernel raises, there is no other path."""
from __future__ import annotations

import torch

from . import _native, kernels, ops


def _blocks(n: int) -> int:
    return -(-n // kernels.FP8_BLOCK)


def _check(name: str, weight: torch.Tensor, scale: torch.Tensor, shape: tuple) -> None:
    want = (*shape[:-2], _blocks(shape[-2]), _blocks(shape[-1]))
    if weight.dtype is not torch.float8_e4m3fn or tuple(weight.shape) != shape:
        raise ValueError(f"{name}: float8_e4m3fn weights {list(shape)} expected, got {weight.dtype} {list(weight.shape)}")
    if not scale.dtype.is_floating_point or tuple(scale.shape) != want:
        raise ValueError(f"{name}: one scale per 128 x 128 block, {list(want)}, expected, got {scale.dtype} {list(scale.shape)}")


def _need_k(name: str, k: int) -> None:
    if k < 16 or k % 16:
        raise ValueError(f"{name}: rows of {k} values; they are fetched in 16-byte pieces, a multiple of 16 is needed")


class BlockFP8Linear(torch.nn.Module):
    """y = quantised(x) . (weight * weight_scale)^T, y of x's type (bf16, fp16 or fp32).  ``load`` takes the checkpoint's
    tensors; ``weight_scale`` multiplies (checkpoints that call it ``weight_scale_inv`` mean the same number)."""

    def __init__(self, in_features: int, out_features: int, *, prefix: str = "block_fp8_linear"):
        super().__init__()
        _need_k(prefix, in_features)
        self.in_features, self.out_features, self.prefix = in_features, out_features, prefix
        self.register_buffer("weight", None)
        self.register_buffer("weight_scale", None)

    def load(self, weight: torch.Tensor, weight_scale: torch.Tensor, device="cuda"):
        _check(self.prefix, weight, weight_scale, (self.out_features, self.in_features))
        _native.load(f"{self.prefix}: block-scaled linear")
        self.weight = weight.to(device).contiguous()
        self.weight_scale = weight_scale.to(device, torch.float32).contiguous()
        _native.prepare(self.weight.device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.weight is None:
            raise RuntimeError(f"{self.prefix}: called before load()")
        if kernels.takes_plan(x):
            return kernels.linear_fp8_blocks(x, self.weight, self.weight_scale, scale_rule=ops.ACT_SCALE_RULE)
        return ops.fp8_blocks_linear(x, self.weight, self.weight_scale)


class BlockFP8MoE(torch.nn.Module):
    """Routed SwiGLU experts: gate and up projections stacked in ``w13`` [E, 2 inter, hidden], the down projection in ``w2``
    [E, hidden, inter], scales of both per 128 x 128 block of the stacked rows.  ``expert_base``: the experts held here are the
    global ids [expert_base, expert_base + E); pairs of others count nothing."""

    def __init__(self, num_experts: int, hidden: int, inter: int, *, expert_base: int = 0, prefix: str = "block_fp8_moe"):
        super().__init__()
        _need_k(prefix, hidden)
        _need_k(prefix, inter)
        if not 1 <= num_experts <= 1024:
            raise ValueError(f"{prefix}: 1 to 1024 experts expected, got {num_experts}")
        self.num_experts, self.hidden, self.inter, self.expert_base, self.prefix = num_experts, hidden, inter, expert_base, prefix
        for name in ("w13", "w13_scale", "w2", "w2_scale"):
            self.register_buffer(name, None)

    def load(self, w13, w13_scale, w2, w2_scale, device="cuda"):
        E, H, I = self.num_experts, self.hidden, self.inter
        _check(f"{self.prefix}.w13", w13, w13_scale, (E, 2 * I, H))
        _check(f"{self.prefix}.w2", w2, w2_scale, (E, H, I))
        _native.load(f"{self.prefix}: block-scaled experts")
        self.w13, self.w2 = w13.to(device).contiguous(), w2.to(device).contiguous()
        self.w13_scale, self.w2_scale = (s.to(device, torch.float32).contiguous() for s in (w13_scale, w2_scale))
        _native.prepare(self.w13.device)
        return self

    def forward(self, x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor) -> torch.Tensor:
        if self.w13 is None:
            raise RuntimeError(f"{self.prefix}: called before load()")
        args = (x, self.w13, self.w13_scale, self.w2, self.w2_scale, topk_weights, topk_ids)
        if kernels.takes_plan(x):
            return kernels.moe_fp8_blocks(*args, expert_base=self.expert_base, scale_rule=ops.ACT_SCALE_RULE)
        return ops.fp8_blocks_moe(*args, self.expert_base)
