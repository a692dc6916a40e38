"""The norms around a residual block, fused with its gate and residual scale.

    u = norm(f) * post_weight + post_bias      the norm after the block f = block(h)
    r = x + scale * gate * u                   the residual stream
    h = norm(r) * pre_weight + pre_bias        the norm before the next block

`norm` is a LayerNorm (kind="layer") or a root-mean-square norm (kind="rms") over the last
axis. One kernel reads x and f and writes r and h; its backward returns the gradients of
x, f, the gate and every parameter in one further pass (csrc/blocknorm.h).

Activations (x, f, gate, r, h) are float32 or bfloat16, one type a call; parameters and
their gradients are float32. Non-contiguous inputs are copied. The last axis holds 1 to
8192 channels.
"""
from __future__ import annotations

import torch
from torch import nn

from . import kern
from ._lib import AccError

KINDS = ("layer", "rms")


def _check(x, f, params, g):
    """Types, devices and sizes; rows P, rows that share a gate L, channels C."""
    kern._check(x, "blocknorm x", act=True)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        raise AccError(f"blocknorm: 1 to 8192 channels on the last axis, got {tuple(x.shape)}")
    C = int(x.shape[-1])
    P = x.numel() // C
    for name, t in (("f", f), ("gate", g)):
        if t is not None and (t.dtype != x.dtype or t.get_device() != x.get_device()):
            raise AccError(f"sandwich_norm {name}: {x.dtype} on {x.device} expected, got "
                           f"{t.dtype} on {t.device}")
    if f is not None and f.shape != x.shape:
        raise AccError(f"sandwich_norm: f {tuple(f.shape)} and x {tuple(x.shape)} differ")
    for name, t in params:
        if t is not None and (t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != C
                              or t.get_device() != x.get_device()):
            raise AccError(f"{name}: float32 [{C}] on {x.device} expected, got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device}")
    L = P
    if g is not None:
        shared = (x.shape[0],) + (1,) * (x.dim() - 2) + (C,) if x.dim() >= 2 else None
        if g.shape == x.shape:
            L = 1
        elif tuple(g.shape) == shared:
            L = P // x.shape[0] if P else 1
        else:
            raise AccError(f"sandwich_norm: gate {tuple(g.shape)} is neither x's shape "
                           f"{tuple(x.shape)} nor one row per sample {shared}")
    return P, L, C


def _apply(*args):
    """Every call goes through the autograd function, one without a backward (`keep`) too:
    forward mode refuses it and a trace records it, where a launch of its own would pass both
    by. Checks and sizes are its own, so a replayed trace has those of its inputs."""
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:8])
    return _BlockNormFn.apply(*args, keep)


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, w1, b1, s, g, w2, b2, layer, eps, want_h, keep):
        pre = "pre_" if f is not None else ""  # norm() has one weight and one bias
        P, L, C = _check(x, f, (("post_weight", w1), ("post_bias", b1), ("scale", s),
                                (pre + "weight", w2), (pre + "bias", b2)), g)
        r = torch.empty_like(x) if f is not None else None
        h = torch.empty_like(x) if want_h else None
        stats = torch.empty(P, 4, dtype=torch.float32, device=x.device) if keep else None
        kern.blocknorm_fwd(x, f, w1, b1, s, g, w2, b2, layer, eps, r, h, stats, P, L, C)
        if keep:
            ctx.save_for_backward(x, f, w1, b1, s, g, w2, stats)
            ctx.cfg = (layer, P, L, C)
            ctx.set_materialize_grads(False)
        return r, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dh):
        x, f, w1, b1, s, g, w2, stats = ctx.saved_tensors
        layer, P, L, C = ctx.cfg
        if dr is None and dh is None:
            return (None,) * 12
        dr = dr.contiguous() if dr is not None else None
        dh = dh.contiguous() if dh is not None else None
        dx = torch.empty_like(x)
        df = torch.empty_like(f) if f is not None else None
        dg = torch.empty_like(g) if g is not None else None
        dpar = torch.empty(5, C, dtype=torch.float32, device=x.device)
        kern.blocknorm_bwd(x, f, w1, b1, s, g, w2, layer, stats, dr, dh, dx, df, dg, dpar, P, L, C)
        par = [d if on else None for d, on in zip(dpar.unbind(0), ctx.needs_input_grad[2:5]
                                                  + ctx.needs_input_grad[6:8])]
        return (dx, df, par[0], par[1], par[2], dg, par[3], par[4]) + (None,) * 4


def _kind(kind):
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {KINDS}, got {kind!r}")
    return kind == "layer"


def _rows(*ts):
    return [None if t is None else t.contiguous() for t in ts]


def sandwich_norm(x, f, post_weight=None, post_bias=None, scale=None, gate=None,
                  pre_weight=None, pre_bias=None, *, kind="layer", eps=1e-5, pre=True):
    """(r, h) of the formulas above; h is None with pre=False (the last block of a model).

    x, f: [..., C]. gate: None, x's shape, or x's shape with every axis but the first and
    the last 1 ([B, 1, ..., C], one row per sample). Weights and scale None mean 1, biases
    None mean 0."""
    layer = _kind(kind)
    if not pre and (pre_weight is not None or pre_bias is not None):
        raise ValueError("sandwich_norm: pre=False takes no pre_weight / pre_bias")
    return _apply(*_rows(x, f, post_weight, post_bias, scale, gate, pre_weight, pre_bias), layer,
                  float(eps), bool(pre))


def norm(x, weight=None, bias=None, *, kind="layer", eps=1e-5):
    """norm(x) * weight + bias over the last axis: the norm before a model's first block."""
    layer = _kind(kind)
    return _apply(*_rows(x, None, None, None, None, None, weight, bias), layer, float(eps), True)[1]


class SandwichNorm(nn.Module):
    """sandwich_norm with its parameters: the norm after a block, the residual scale
    (started at `scale_init`, None for no scale) and the norm before the next block
    (pre=False: none)."""

    def __init__(self, dim, kind="layer", eps=1e-5, bias=True, scale_init=1.0, pre=True):
        super().__init__()
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {KINDS}, got {kind!r}")
        self.kind, self.eps, self.pre = kind, eps, pre

        def par(value, on=True):
            return nn.Parameter(torch.full((dim,), float(value))) if on else None

        self.post_weight, self.post_bias = par(1), par(0, bias)
        self.scale = par(scale_init) if scale_init is not None else None
        self.pre_weight, self.pre_bias = par(1, pre), par(0, pre and bias)

    def forward(self, x, f, gate=None):
        return sandwich_norm(x, f, self.post_weight, self.post_bias, self.scale, gate,
                             self.pre_weight, self.pre_bias, kind=self.kind, eps=self.eps,
                             pre=self.pre)
