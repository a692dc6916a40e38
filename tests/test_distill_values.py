"""Distillation (accunet/distill.py): logits far from zero or masked with the type's lowest
value, and classes listed more than once, against the definition in 64 bits on distributions
over all classes.

Tolerance, u = 2^-24, e the exponent (z - m) * log2(e) / T of a softmax term: the difference,
the factor and the product round once each, so 2^e is off by 3 u |e| ln 2 + 2 u (exp2); the
largest logits of a thread, a wave, a block and the row are joined over such factors four
times; a sum is at most 64 additions in turn and 12 in a tree; a gradient multiplies three more
values. The teacher's K masses are formed the same way and added up where their class is the
same. So a probability is off by at most (9 D + 100 + K) u of itself, D the largest |e|, and the
loss by that share of sum p (|log p| + |log q| + 1). None of it depends on where the logits lie.
Terms below 2^-126 are stored as zero, so D counts up to 150. bf16 gradients add half a step."""
import math

import pytest
import torch

from accunet import _lib
from test_distill import NEG, U, _close, _fn, _hard, _make


def _exact(z, idx, top, rest, T):
    """Loss and gradient (unit upstream) a row, [R][V], and their bounds."""
    z, top = z.double(), top.double()
    R, V = z.shape
    ok = (idx >= 0) & (idx < V)
    live = (ok & (top > NEG)).any(1)
    t = torch.where(ok, top / T, torch.full_like(top, NEG))
    t = torch.where(live[:, None], t, torch.zeros_like(t))
    r = rest.double() if rest is not None else torch.zeros(R, dtype=torch.float64)
    at = torch.where(ok, idx, torch.zeros_like(idx)).long()
    each = torch.where(ok, torch.softmax(t, 1) * (1 - r)[:, None], torch.zeros_like(t))
    p = torch.zeros_like(z).scatter_add_(1, at, each)  # entries of one class add up
    mask = torch.zeros_like(z).scatter_add_(1, at, ok.double()) > 0
    lq = torch.log_softmax(z / T, 1)
    q = lq.exp()
    on = p > 0
    lp = torch.log(torch.where(on, p, torch.ones_like(p)))
    lq_on = torch.where(on, lq, torch.zeros_like(lq))
    loss = (p * (lp - lq_on)).sum(1)
    mag = (p * (lp.abs() + lq_on.abs() + 1)).sum(1)
    d, m = q - p, q + p
    if rest is not None:
        lr = torch.logsumexp(lq.masked_fill(mask, NEG), 1)
        some = (r > 0) & (lr > NEG)
        lr0, r0 = torch.where(some, lr, torch.zeros_like(lr)), torch.where(some, r, torch.zeros_like(r))
        lr_r = torch.log(torch.where(some, r, torch.ones_like(r)))
        loss, mag = loss + r0 * (lr_r - lr0), mag + r0 * (lr_r.abs() + lr0.abs() + 1)
        share = torch.where(mask, torch.zeros_like(q), (lq - lr0[:, None]).exp()) * r0[:, None]
        d, m = d - share, m + share
    fin = torch.isfinite(z)
    hi = torch.where(fin, z, torch.full_like(z, NEG)).amax(1)
    lo = torch.where(fin, z, torch.full_like(z, math.inf)).amin(1)
    has = ok & (top > NEG)
    spread = (torch.where(has, top, torch.full_like(top, NEG)).amax(1)
              - torch.where(has, top, torch.full_like(top, math.inf)).amin(1))
    D = (torch.maximum(hi - lo, spread) / T * 1.4427).clamp(min=0.0, max=150.0)
    k = (9 * D + 100 + idx.shape[1]) * U
    z0 = torch.zeros((), dtype=torch.float64)
    loss, mag = torch.where(live, loss, z0) * T * T, torch.where(live, mag, z0) * T * T
    d, m = torch.where(live[:, None], d, z0) * T, torch.where(live[:, None], m, z0) * T
    return loss, d, k * mag, k[:, None] * m, live


def _compare(z, idx, top, r, T, planes=None):
    """One loss a row and the mean, with their gradients; planes: (B, S)."""
    want, dwant, tl, td, live = _exact(z, idx, top, r, T)
    dev = [t.cuda() if t is not None else None for t in (z, idx, top, r)]
    dim = -1
    if planes:
        B, S = planes
        dev[:3] = [t.view(B, S, -1).movedim(-1, 1).contiguous() for t in dev[:3]]
        dev[3] = dev[3].view(B, S) if r is not None else None
        dim = 1
    zd = dev[0].requires_grad_()
    for reduction, n in (("none", 1), ("mean", max(1, int(live.sum())))):
        loss = _fn()(zd, dev[1], dev[2], rest=dev[3], temperature=T, reduction=reduction, dim=dim)
        (dz,) = torch.autograd.grad(loss, zd, torch.ones_like(loss))
        if planes:
            dz = dz.movedim(1, -1).reshape(z.shape)
        if reduction == "none":
            _close(loss.reshape(-1), want, tl, "loss")
        else:
            _close(loss, want.sum() / n, (tl.sum() + 8 * U * want.abs().sum()) / n, "mean")
        _close(dz, dwant / n, (td + 8 * U * dwant.abs()) / n, f"dz {reduction}")


# a row in registers; a row cut over blocks; one block a row; images
LAYOUTS = [(6, 257, 9, None), (5, 5003, 17, None), (260, 2500, 5, None), (12, 12, 4, (2, 6)),
           (10, 150, 20, (2, 5))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,K,planes", LAYOUTS)
@pytest.mark.parametrize("offset", [1e4, -1e4, 3e5])
def test_logits_far_from_zero(R, V, K, planes, offset, dtype):
    for i, rest in enumerate((False, True)):
        z, idx, top, r = _make(R, V, K, torch.float32, rest, seed=20 + i)
        _compare((z + offset).to(dtype), idx, (top - offset).to(dtype), r, 2.0, planes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,K,planes", LAYOUTS)
@pytest.mark.parametrize("T", [1.0, 0.5])
def test_classes_masked_with_the_lowest_value(R, V, K, planes, T, dtype):
    """The first half of the classes masked (whole vectors of a thread, whole groups of a
    pixel), every class of a row, and every entry of the teacher, at the lowest value and at
    -inf: a softmax over equal logits is uniform, wherever they lie."""
    lowest = torch.finfo(dtype).min
    for i, rest in enumerate((False, True)):
        z, idx, top, r = _make(R, V, K, dtype, rest, seed=30 + i)
        g = torch.Generator().manual_seed(40 + i)
        idx = V // 2 + torch.rand(R, V - V // 2, generator=g).argsort(1)[:, :K]
        z[:, :V // 2] = lowest
        z[1, :V // 2] = NEG
        z[2] = lowest
        top[3] = lowest
        top[4, 1:] = lowest
        if rest:
            # where the classes outside the entries are masked, the teacher has no mass there
            r[torch.isinf(z).any(1)] = 0.0
            free = torch.ones(R, V, dtype=torch.bool).scatter_(1, idx, False)
            r[~(free & (z > lowest)).any(1) & (torch.arange(R) != 2)] = 0.0
        _compare(z, idx, top, r, T, planes)


REPEATED = [(8, 7, 3, None), (9, 40, 6, None), (7, 257, 200, None), (6, 5003, 256, None),
            (260, 2500, 9, None), (12, 12, 4, (2, 6)), (10, 150, 70, (2, 5))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,K,planes", REPEATED)
def test_repeated_entries_add_up(R, V, K, planes, dtype):
    """p log p is taken of a class's whole mass, however many entries it is split over."""
    for i, rest in enumerate((False, True)):
        z, _, top, r = _make(R, V, 1, dtype, rest, seed=50 + i)
        g = torch.Generator().manual_seed(60 + i)
        idx = torch.randint(0, max(2, min(V, K // 2)), (R, K), generator=g)
        top = (2 * torch.randn(R, K, generator=g)).to(dtype)
        idx[0] = V - 1                   # one class
        idx[1, ::2] = -1                 # padding between the entries
        top[2, :K // 2] = NEG            # entries of no mass beside others of their class
        idx[3], top[3, 1:] = 1, NEG      # a class's first entry has all its mass
        idx[4], top[4, :-1] = 1, NEG     # its last one
        top[5] = torch.linspace(-60, 0, K).to(dtype)  # masses of very different size
        _compare(z, idx, top, r, 1.7, planes)


@pytest.mark.gpu
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("V", [30, 900])
@pytest.mark.parametrize("K", [2, 3, 65, 256])
def test_a_certain_student_has_no_loss(K, V, planes):
    """Equal entries of one class, of which the student is certain: the distributions are the
    same, so loss and gradient are zero. K masses of 1 / K add up to 1 within K u, and
    log2 1 is 0; the student's other classes have 2^-140 of its mass at most."""
    z = torch.full((4, V, 3) if planes else (4, V), -100.0, device="cuda")
    shape = (4, K, 3) if planes else (4, K)
    z[:, 5] = 0.0
    z.requires_grad_()
    idx = torch.full(shape, 5, device="cuda")
    loss = _fn()(z, idx, torch.zeros(shape, device="cuda"), temperature=1.0, reduction="sum", dim=1)
    (dz,) = torch.autograd.grad(loss, z)
    assert abs(float(loss.detach())) <= 12 * (2 * K + 4) * U and float(dz.abs().max()) <= (2 * K + 4) * U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,K,planes", [(40, 6, None), (40, 6, (2, 7)), (3001, 70, None),
                                        (1000, 70, (2, 7))])
def test_hard_rows(V, K, dtype, planes):
    """The rows of test_distill.py's _hard, among them one that lists a class many times."""
    z, idx, top, r = _hard(V, K, dtype)
    for rest in (r, None):
        _compare(z, idx, top, rest, 1.7, planes)
    z[7, idx[7, 0]] = 0.0  # every loss finite
    for rest in (r, None):
        _compare(z, idx, top, rest, 1.7, planes)


def test_temperatures_whose_square_leaves_fp32_are_refused():
    """The loss is multiplied by T^2, its exponents by log2(e) / T: beyond 2^-60 and 2^60 one of
    them overflowed or became zero, and with it the loss (NaN, or zero for a positive one)."""
    z, i, t = torch.zeros(2, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for bad in (1e-45, 1e-39, 2.0 ** -61, 2.0 ** 61, 1e30, 1e39):
        with pytest.raises(ValueError):
            _fn()(z, i, t, temperature=bad)
    lib = _lib.load()
    n, m = lib.accunet_distill_save_bytes(2, 1, 5, 3), lib.accunet_distill_ws_bytes(2, 1, 5, 3, 0)
    for bad in (1e-39, 2.0 ** -61, 2.0 ** 61, 1e30):
        assert lib.accunet_distill_fwd(16, 16, 1, 16, 0, None, 16, 2, None, 16, n, 16, m, 2, 1, 5, 3,
                                       bad, 1.0, 0, None) == -2
        assert lib.accunet_distill_bwd(16, 16, n, 16, 2, 0, 16, 2, 1, 5, 3, bad, 1.0, 0, None) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60])
def test_extreme_temperatures(T):
    """Logits of the size of T, so that the distributions are ordinary ones."""
    z, idx, top, r = _make(5, 300, 6, torch.float32, True, seed=70)
    _compare(z * T, idx, top * T, r, T)
