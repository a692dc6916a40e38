"""Distillation loss from a teacher's top logits, with its gradient.

A stored teacher answer is K class indices and logits a row (a token, a pixel) and, if
kept, the probability mass outside them. With p the teacher's softmax over its entries
(scaled by 1 - rest) and q the student's softmax over all V classes, both at the
temperature T:

    loss = weight * T^2 * [ sum_k p_k (log p_k - log q_k) + rest (log rest - log q_rest) ]

q_rest is the student's mass outside the entries; without `rest` the teacher has no mass
there. The gradient is that of the student's logits (csrc/distill.h).

Rows: an entry whose index lies outside [0, V) is padding, entries of the same class add
up, an entry whose logit is -inf has no mass. A row without a valid entry has loss 0 and
gradient 0 and does not count in the mean. A student logit of -inf is a class of
probability 0 (infinite loss where the teacher has mass there).
"""
from __future__ import annotations

import math

import torch

from . import kern
from ._lib import AccError

MAX_K = 256
_PLANES_MAX_V = 1024
_MIN_T = 2.0 ** -60  # T^2 and 1 / T are normal float32 numbers
_REDUCTIONS = ("none", "sum", "mean")


def _sizes(z, idx, top, rest, planes):
    """Checks; B, S, V, K of the kernels (rows: B of them, S = 1)."""
    kern._check(z, "topk_distill logits", act=True)
    axis, shape = 1 if planes else z.dim() - 1, tuple(z.shape)
    V, K = int(shape[axis]), (int(idx.shape[axis]) if idx.dim() == z.dim() else 0)
    want, outer = shape[:axis] + (K,) + shape[axis + 1:], shape[:axis] + shape[axis + 1:]
    if not 1 <= K <= MAX_K or tuple(idx.shape) != want or tuple(top.shape) != want:
        raise AccError(f"topk_distill: top_idx {tuple(idx.shape)} and top_logits "
                       f"{tuple(top.shape)} must have 1 to {MAX_K} entries in place of "
                       f"the {V} classes of {shape}")
    if not 1 <= V <= 1 << 30:
        raise AccError(f"topk_distill: 1 to 2^30 classes, got {V}")
    if idx.dtype not in (torch.int32, torch.int64):
        raise AccError(f"topk_distill: int32 or int64 top_idx, got {idx.dtype}")
    kern._check(top, "topk_distill top_logits", act=True)
    if rest is not None:
        kern._check(rest, "topk_distill rest")
        if tuple(rest.shape) != outer:
            raise AccError(f"topk_distill: rest {tuple(rest.shape)}, expected {outer}")
    for name, t in (("top_idx", idx), ("top_logits", top), ("rest", rest)):
        if t is not None and t.device != z.device:
            raise AccError(f"topk_distill: {name} on {t.device}, logits on {z.device}")
    n = 1
    for s in outer:
        n *= int(s)
    B = int(shape[0]) if planes else n
    return B, (n // B if B else 0) if planes else 1, V, K, outer


class _DistillFn(torch.autograd.Function):
    """The forward writes the gradient for an upstream of 1 where one kernel can do both
    (sum and mean), and the backward hands that tensor out, once: its kernel rewrites it only
    for another upstream gradient. A further backward of the same graph computes it anew, and
    so does a backward in another graph capture than the forward's: replayed by itself, it
    would hand out what the consumers of the last replay left in that tensor.

    Every call goes through here, one without a backward (`grad`) too: forward mode refuses it
    and a trace records it, where a launch of its own would pass both by. Checks and sizes are
    its own, so a replayed trace has those of its inputs."""

    @staticmethod
    def forward(ctx, z, idx, top, rest, T, weight, reduction, planes, grad):
        B, S, V, K, outer = _sizes(z, idx, top, rest, planes)
        new = torch.empty if B * S else torch.zeros
        loss = new(outer if reduction == 0 else (), dtype=torch.float32, device=z.device)
        if z.data_ptr() % 16:
            z = z.clone()
        dz = save = None
        if grad and reduction != 0 and B * S and kern.distill_fused(B, S, V, kern._dt(z)):
            dz = torch.empty_like(z)
        if B * S:
            save = kern.distill_fwd(z, idx, top, rest, loss, reduction, dz, B, S, V, K, T, weight)
        if grad:
            ctx.dz, ctx.capture = dz, kern.capture_id(z)
            ctx.save_for_backward(z, save)
            ctx.cfg = (reduction, B, S, V, K, T, weight)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        z, save = ctx.saved_tensors
        dz, ctx.dz = ctx.dz, None
        held = dz is not None and ctx.capture == kern.capture_id(z) >= 0
        if not held:
            dz = torch.empty_like(z)
        if save is not None:
            reduction, B, S, V, K, T, weight = ctx.cfg
            kern.distill_bwd(z, save, up.contiguous(), reduction, held, dz, B, S, V, K, T, weight)
        return (dz,) + (None,) * 8


def topk_distill(logits, top_idx, top_logits, rest=None, temperature=1.0, weight=1.0,
                 reduction="mean", dim=-1):
    """The loss of the module docstring.

    logits: [..., V] (dim=-1) or [B, V, ...] (dim=1), float32 or bfloat16. top_idx (int32 or
    int64) and top_logits (float32 or bfloat16): the same shape with K <= 256 entries in
    place of the V classes. rest: float32, the shape without that axis, in [0, 1].
    reduction: "mean" over the rows that have an entry, "sum", or "none" (one loss a row).
    temperature: 2^-60 to 2^60.
    `weight` multiplies the loss (inside: a factor applied to the result, 0.5 * loss, costs the
    backward another pass over the logits). Non-contiguous inputs are copied, and so are more than
    1024 classes on dim=1. At most 2^26 - 4 rows with the classes last, 2^24 - 1 above 2032
    classes."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    temperature, weight = float(temperature), float(weight)
    if not _MIN_T <= temperature <= 1 / _MIN_T:
        raise ValueError(f"temperature must lie between 2^-60 and 2^60, got {temperature}")
    nd = logits.dim()
    axis = dim + nd if dim < 0 else dim
    if nd < 1 or axis not in (nd - 1, 1) or not 0 <= axis < nd:
        raise AccError(f"topk_distill: the classes lie on the last axis or on axis 1, got "
                       f"dim={dim} of {tuple(logits.shape)}")
    for name, t in (("top_idx", top_idx), ("top_logits", top_logits), ("rest", rest)):
        if t is not None and t.requires_grad:
            raise ValueError(f"topk_distill: no gradient flows to {name}; detach it")
    args = (logits, top_idx, top_logits)
    planes = axis != nd - 1
    if planes and (logits.shape[1] > _PLANES_MAX_V or math.prod(logits.shape[2:]) <= 1):
        # too many classes, or one pixel a sample (no copy then)
        args = [t.movedim(axis, -1) if t.dim() == nd else t for t in args]
        planes = False
    return _DistillFn.apply(*(t.contiguous() for t in args),
                            rest.contiguous() if rest is not None else None, temperature, weight,
                            _REDUCTIONS.index(reduction), planes,
                            torch.is_grad_enabled() and logits.requires_grad)
