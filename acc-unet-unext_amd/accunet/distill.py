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

import torch

from . import kern
from ._lib import AccError

MAX_K = 256
_PLANES_MAX_V = 1024
_REDUCTIONS = ("mean", "sum", "none")


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, idx, top, rest, T, weight, reduction, B, S, V, K, planes):
        dev = z.device
        n = B * S
        f32 = torch.float32
        none = reduction == "none"
        if n == 0:
            ctx.empty = True
            ctx.like = z.shape, z.dtype
            return torch.zeros((0,) if none else (), dtype=f32, device=dev)
        ctx.empty = False
        id_ = torch.empty(n * K, dtype=torch.int32, device=dev)
        p = torch.empty(n * K, dtype=f32, device=dev)
        tea = torch.empty(n, 2, dtype=f32, device=dev)
        state = torch.empty(n, 4, dtype=f32, device=dev)
        count = torch.zeros(1, dtype=torch.int32, device=dev)
        kern.distill_teacher(idx, top, rest, id_, p, tea, count, B, S, V, K, T)
        rowloss = torch.empty(n, dtype=f32, device=dev) if none else None
        nb = (n + 255) // 256 if planes else n
        part = torch.empty(nb, dtype=torch.float64, device=dev)
        kern.distill_fwd(z, rest, id_, p, tea, state, rowloss, part, B, S, V, K, T, weight, planes)
        if not none:
            loss = torch.empty((), dtype=f32, device=dev)
            kern.distill_loss(part, nb, count if reduction == "mean" else None, loss)
        ctx.save_for_backward(z, id_, p, state, count)
        ctx.cfg = (T, weight, reduction, B, S, V, K, planes)
        return rowloss if none else loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        if ctx.empty:
            shape, dtype = ctx.like
            return (torch.zeros(shape, dtype=dtype, device=up.device),) + (None,) * 11
        z, id_, p, state, count = ctx.saved_tensors
        T, weight, reduction, B, S, V, K, planes = ctx.cfg
        dz = torch.empty_like(z)
        kern.distill_bwd(z, id_, p, state, up.contiguous(), reduction == "none",
                         count if reduction == "mean" else None, dz, B, S, V, K, T, weight, planes)
        return (dz,) + (None,) * 11


def topk_distill(logits, top_idx, top_logits, rest=None, temperature=1.0, weight=1.0,
                 reduction="mean", dim=-1):
    """The loss of the module docstring.

    logits: [..., V] (dim=-1) or [B, V, ...] (dim=1), float32 or bfloat16. top_idx (int32 or
    int64) and top_logits (float32 or bfloat16): the same shape with K <= 256 entries in
    place of the V classes. rest: float32, the shape without that axis, in [0, 1].
    reduction: "mean" over the rows that have an entry, "sum", or "none" (one loss a row).
    `weight` multiplies the loss. Non-contiguous inputs are copied, and so are more than
    1024 classes on dim=1."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    temperature, weight = float(temperature), float(weight)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    kern._check(logits, "topk_distill logits", act=True)
    nd = logits.dim()
    axis = dim + nd if dim < 0 else dim
    if nd < 1 or axis not in (nd - 1, 1) or not 0 <= axis < nd:
        raise AccError(f"topk_distill: the classes lie on the last axis or on axis 1, got "
                       f"dim={dim} of {tuple(logits.shape)}")
    shape = list(logits.shape)
    V, K = shape[axis], (top_idx.shape[axis] if top_idx.dim() == nd else 0)
    want = shape[:axis] + [K] + shape[axis + 1:]
    outer = shape[:axis] + shape[axis + 1:]
    if not 1 <= K <= MAX_K or list(top_idx.shape) != want or list(top_logits.shape) != want:
        raise AccError(f"topk_distill: top_idx {tuple(top_idx.shape)} and top_logits "
                       f"{tuple(top_logits.shape)} must have 1 to {MAX_K} entries in place of "
                       f"the {V} classes of {tuple(shape)}")
    if not 1 <= V <= 1 << 30:
        raise AccError(f"topk_distill: 1 to 2^30 classes, got {V}")
    if top_idx.dtype not in (torch.int32, torch.int64):
        raise AccError(f"topk_distill: int32 or int64 top_idx, got {top_idx.dtype}")
    kern._check(top_logits, "topk_distill top_logits", act=True)
    if rest is not None:
        kern._check(rest, "topk_distill rest")
        if list(rest.shape) != outer:
            raise AccError(f"topk_distill: rest {tuple(rest.shape)}, expected {tuple(outer)}")
    for name, t in (("top_idx", top_idx), ("top_logits", top_logits), ("rest", rest)):
        if t is not None and t.device != logits.device:
            raise AccError(f"topk_distill: {name} on {t.device}, logits on {logits.device}")
        if t is not None and t.requires_grad:
            raise ValueError(f"topk_distill: no gradient flows to {name}; detach it")
    S = 1
    for s in shape[axis + 1:]:
        S *= s
    planes = axis != nd - 1 and S > 1
    if planes and V > _PLANES_MAX_V:
        logits, top_idx, top_logits = (t.movedim(axis, -1) for t in (logits, top_idx, top_logits))
        planes = False
    B = 1
    for s in (shape[:axis] if planes else outer):
        B *= s
    z = logits.contiguous()
    if z.data_ptr() % 16:
        z = z.clone()
    loss = _DistillFn.apply(z, top_idx.contiguous(), top_logits.contiguous(),
                            rest.contiguous() if rest is not None else None, temperature, weight,
                            reduction, B, S if planes else 1, V, K, planes)
    return loss.view(outer) if reduction == "none" else loss
