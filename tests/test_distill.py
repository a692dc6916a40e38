"""Distillation from a teacher's top logits (accunet/distill.py) against its definition in
64 bits, written as distributions over all classes.

Tolerance: with u = 2^-24 a softmax term 2^(z*c - m*c) is off by 2u times its exponent (the
rounding of c and of m*c) plus u of the fma and 2u of exp2; sums are trees over at most 64
successive terms a thread. So q is off by at most 64 * u * (4 + D) relative, D the largest
difference of finite logits over T in base 2, and the loss by that share of
sum p (|log p| + |log q| + 1); bf16 gradients add half a step, eps / 2 of the value. A
gradient below the normal range of fp32 (and bf16) may be flushed to zero: 2^-126 on top."""
import math

import pytest
import torch

from accunet import _lib

U = 2.0 ** -24
NEG = -math.inf


def _fn():
    from accunet.distill import topk_distill
    return topk_distill


# ---------------------------------------------------------------------- refusals (CPU)
def test_refusals_on_the_host():
    f = _fn()
    z, i, t = torch.zeros(2, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    with pytest.raises(_lib.AccError):
        f(z, i, t)  # host tensors
    with pytest.raises(ValueError):
        f(z, i, t, reduction="batch")
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            f(z, i, t, temperature=bad)
    lib = _lib.load()
    ok = 16
    fwd, bwd = lib.accunet_distill_fwd, lib.accunet_distill_bwd

    def f_(R=2, S=1, V=5, K=3, T=1.0, dt=0, red=2, dz=None, z=ok, top_dt=0, short=0, save=16):
        n, m = lib.accunet_distill_save_bytes(2, 1, 5, 3), lib.accunet_distill_ws_bytes(2, 1, 5, 3, 0)
        return fwd(z, ok, 1, ok, top_dt, None, ok, red, dz, save, n - short, ok, m, R, S, V, K, T,
                   1.0, dt, None)

    assert f_(K=257) == -1 and f_(R=0) == -1 and f_(S=9, V=1025) == -1 and f_(V=0) == -1
    assert f_(top_dt=2) == -2 and f_(dt=2) == -2 and f_(T=0.0) == -2 and f_(red=3) == -2
    assert f_(z=None) == -2 and f_(short=1) == -2 and f_(save=8) == -2
    assert f_(dz=24) == -2 and f_(dz=16, red=0) == -2   # dz at another address modulo 16; no sum
    n = lib.accunet_distill_save_bytes(3, 1, 100, 4)
    assert bwd(16, ok, n, ok, 2, 0, 24, 3, 1, 100, 4, 1.0, 1.0, 0, None) == -2  # addresses
    assert bwd(16, ok, n - 1, ok, 2, 0, 16, 3, 1, 100, 4, 1.0, 1.0, 0, None) == -2
    assert bwd(16, ok, n, ok, 0, 1, 16, 3, 1, 100, 4, 1.0, 1.0, 0, None) == -2  # held, no sum
    # a few long rows are cut over blocks: no gradient in the forward
    assert lib.accunet_distill_fused(3, 1, 50021, 0) == 0
    assert lib.accunet_distill_fused(300, 1, 50021, 0) == 1
    assert lib.accunet_distill_fused(3, 1, 2048, 0) == 1 and lib.accunet_distill_fused(2, 9, 5, 0) == 1


def test_more_rows_than_a_launch_holds_are_refused():
    """A launch holds fewer than 2^32 threads: 64 for a row, 256 for one of more than 2032
    classes; pixels of a plane take one each."""
    lib = _lib.load()
    for V, most in ((9, 2 ** 26 - 4), (2032, 2 ** 26 - 4), (2033, 2 ** 24 - 1)):
        assert lib.accunet_distill_save_bytes(most, 1, V, 1) > 0
        assert lib.accunet_distill_save_bytes(most + 1, 1, V, 1) == 0
        assert lib.accunet_distill_ws_bytes(most + 1, 1, V, 1, 0) == 0
        assert lib.accunet_distill_fwd(16, 16, 1, 16, 0, None, 16, 2, None, 16, 2 ** 62, 16, 2 ** 62,
                                       most + 1, 1, V, 1, 1.0, 1.0, 0, None) == -1
        assert lib.accunet_distill_bwd(16, 16, 2 ** 62, 16, 2, 0, 16, most + 1, 1, V, 1, 1.0, 1.0,
                                       0, None) == -1
    assert lib.accunet_distill_save_bytes(1, 2 ** 31 - 1, 9, 1) > 0
    assert lib.accunet_distill_save_bytes(1, 2 ** 31, 9, 1) == 0


# ----------------------------------------------------------------------- the reference
def _reference(z, idx, top, rest, T, weight=1.0):
    """Per-row loss and gradient (unit upstream) in 64 bits, rows [R][V], with bounds."""
    z, top = z.double(), top.double()
    R, V = z.shape
    ok = (idx >= 0) & (idx < V)
    live = (ok & ~(top == NEG)).any(1)
    loss, dz = torch.zeros(R, dtype=torch.float64), torch.zeros(R, V, dtype=torch.float64)
    tl, td = torch.zeros_like(loss), torch.zeros_like(dz)
    for i in range(R):
        if not live[i]:
            continue
        ids, tt = idx[i][ok[i]], top[i][ok[i]]
        r = float(rest[i]) if rest is not None else 0.0
        pk = torch.softmax(tt / T, 0) * (1.0 - r)
        p = torch.zeros(V, dtype=torch.float64).index_add_(0, ids, pk)
        mask = torch.zeros(V, dtype=torch.bool)
        mask[ids] = True
        lq = torch.log_softmax(z[i] / T, 0)
        a = pk > 0
        terms = pk[a] * (torch.log(pk[a]) - lq[ids][a])
        mags = pk[a] * (torch.log(pk[a]).abs() + lq[ids][a].abs() + 1)
        q = lq.exp()
        d = q - p
        m = q + p
        extra = em = 0.0
        if rest is not None:
            lr = torch.logsumexp(lq.masked_fill(mask, NEG), 0)
            if r > 0:
                extra = r * (math.log(r) - float(lr))
                em = r * (abs(math.log(r)) + abs(float(lr)) + 1)
                if lr > NEG:
                    share = torch.where(mask, torch.zeros_like(q), (lq - lr).exp())
                    d, m = d - r * share, m + r * share
        fin = z[i][torch.isfinite(z[i])]
        D = float((fin.max() - fin.min()) / T) * 1.4427 if fin.numel() else 0.0
        k = 64 * U * (4 + D)
        loss[i] = weight * T * T * (terms.sum() + extra)
        tl[i] = k * weight * T * T * (mags.sum() + em)
        dz[i], td[i] = weight * T * d, k * weight * T * m
    return loss, dz, tl, td, live


def _make(R, V, K, dtype, rest, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (spread * torch.randn(R, V, generator=g)).to(dtype)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)])
    top = (2 * torch.randn(R, K, generator=g)).to(dtype)
    r = torch.rand(R, generator=g) * 0.6 if rest else None
    if rest and K == V:
        r.zero_()
    return z, idx, top, r


def _close(got, want, tol, name):
    got = got.detach().cpu()
    tol = tol + 2.0 ** -126  # a magnitude below it stored as zero is off by less than that
    if got.dtype == torch.bfloat16:
        tol = tol + want.abs() * torch.finfo(torch.bfloat16).eps / 2 * (1 + 2 ** -8)
    both_inf = (want == got.double()) & torch.isinf(want)
    over = torch.where(both_inf, torch.zeros_like(want), (got.double() - want).abs() - tol)
    assert float(over.max()) <= 0, (name, float(over.max()))


def _check(z, idx, top, r, T=1.7, weight=1.0, reduction="mean", planes=None, **kw):
    """planes: (B, S) lays the rows out as [B, V, S]."""
    loss64, dz64, tl, td, live = _reference(z, idx, top, r, T, weight)
    dev = [t.cuda() if t is not None else None for t in (z, idx, top, r)]
    dim = -1
    if planes:
        B, S = planes
        dev[:3] = [t.view(B, S, -1).movedim(-1, 1).contiguous() for t in dev[:3]]
        dev[3] = dev[3].view(B, S) if r is not None else None
        dim = 1
    zd = dev[0].requires_grad_()
    loss = _fn()(zd, dev[1], dev[2], rest=dev[3], temperature=T, weight=weight,
                 reduction=reduction, dim=dim)
    up = torch.full_like(loss, 0.75) if reduction != "none" else torch.rand_like(loss) + 0.5
    (dz,) = torch.autograd.grad(loss, zd, up)
    if planes:
        dz = dz.movedim(1, -1).reshape(z.shape)
    n = max(1, int(live.sum())) if reduction == "mean" else 1
    up = up.detach().double().cpu().reshape(-1)
    if reduction == "none":
        _close(loss.reshape(-1), loss64, tl, "loss")
        f = up[:, None]
    else:
        _close(loss, loss64.sum() / n, tl.sum() / n + 8 * U * (loss64.sum() / n).abs(), "loss")
        f = up / n
    _close(dz, dz64 * f, (td + 8 * U * dz64.abs()) * f, "dz")
    return loss, dz


ROWS = [(1, 1, 1), (3, 2, 1), (5, 7, 7), (9, 33, 5), (4, 257, 64), (6, 2048, 100), (3, 2049, 256),
        (2, 5003, 17), (1, 70001, 64), (2, 140003, 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", ROWS)
def test_rows_match_64_bits(shape, dtype):
    for i, rest in enumerate((False, True)):
        _check(*_make(*shape, dtype, rest, seed=i))
    _check(*_make(*shape, dtype, True, seed=7), reduction="none", weight=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,V,K", [(1, 2, 2, 1), (2, 257, 3, 3), (3, 100, 12, 4), (1, 300, 33, 8),
                                     (2, 40, 150, 20), (1, 70, 1024, 3), (1, 30, 1025, 3)])
def test_planes_match_64_bits(B, S, V, K, dtype):
    for i, rest in enumerate((False, True)):
        _check(*_make(B * S, V, K, dtype, rest, seed=i), planes=(B, S))
    _check(*_make(B * S, V, K, dtype, True, seed=7), planes=(B, S), reduction="none")
    _check(*_make(B * S, V, K, dtype, False, seed=8), planes=(B, S), reduction="sum", T=1.0)


def _hard(V, K, dtype):
    """Rows where it can go wrong: see the comments."""
    z, idx, top, r = _make(14, V, K, dtype, True, seed=11)
    idx[0] = -1                               # no entry at all
    idx[1] = V                                # every index past the classes
    top[2] = NEG                              # entries, but no mass
    idx[3, 1:] = -1                           # one entry left
    idx[4, K // 2:] = idx[4, 0]               # the same class many times
    top[5, 1:] = NEG                          # entries of no mass are still listed
    z[6] = NEG                                # masked classes of the student
    z[6, idx[6]] = 1.0
    r[6] = 0.0
    z[7, idx[7, 0]] = NEG                     # the teacher's mass on a masked class: infinite
    z[8, idx[8]] = 200.0                      # q_rest below fp32's range
    z[9] = torch.finfo(torch.bfloat16).min    # masked with the type's lowest value
    z[9, idx[9]] = 0.5
    r[9] = 0.0
    z[0] = math.nan                           # ignored rows may hold anything
    z[1] = math.inf
    r[10] = 1.0                               # all mass outside
    r[11] = 0.0
    z[12] = 5.0                               # equal logits
    top[12] = 1.0
    z[13] -= 1000.0
    return z, idx, top, r


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,K", [(40, 6), (3001, 70)])
@pytest.mark.parametrize("planes", [False, True])
def test_hard_rows(V, K, dtype, planes):
    z, idx, top, r = _hard(V, K, dtype)
    if planes and V > 1024:
        V = 1000
        z, idx, top, r = _hard(V, K, dtype)
    pl = (2, 7) if planes else None
    loss, dz = _check(z, idx, top, r, reduction="none", planes=pl)
    flat = loss.detach().reshape(-1).cpu()
    assert (flat[:3] == 0).all() and torch.equal(dz[:3].cpu(), torch.zeros_like(z[:3]))
    assert math.isinf(float(flat[7])) and bool(torch.isfinite(dz[3:].float()).all())
    z[7, idx[7, 0]] = 0.0
    _check(z, idx, top, r, reduction="mean", planes=pl)
    # without a remaining mass
    _check(z, idx, top, None, reduction="none", planes=pl)


@pytest.mark.gpu
def test_nan_reaches_the_loss():
    z, idx, top, r = _make(3, 50, 4, torch.float32, True)
    z[1, 7] = math.nan
    loss = _fn()(z.cuda(), idx.cuda(), top.cuda(), rest=r.cuda(), reduction="none").cpu()
    assert math.isnan(float(loss[1])) and torch.isfinite(loss[[0, 2]]).all()
    top[2, 1] = math.nan
    loss = _fn()(z.cuda(), idx.cuda(), top.cuda(), rest=r.cuda(), reduction="none").cpu()
    assert math.isnan(float(loss[2])) and math.isfinite(float(loss[0]))


@pytest.mark.gpu
def test_no_rows_and_no_counted_rows():
    f = _fn()
    z = torch.randn(0, 8, device="cuda", requires_grad=True)
    loss = f(z, torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda"))
    loss.backward()
    assert float(loss) == 0.0 and z.grad.shape == (0, 8)
    z = torch.randn(3, 8, device="cuda", requires_grad=True)
    loss = f(z, torch.full((3, 2), -1, device="cuda"), torch.zeros(3, 2, device="cuda"))
    loss.backward()
    assert float(loss) == 0.0 and torch.equal(z.grad, torch.zeros_like(z))


@pytest.mark.gpu
def test_types_strides_and_module():
    from accunet.loss import TopKDistill
    f = _fn()
    z, idx, top, r = (t.cuda() for t in _make(12, 700, 9, torch.bfloat16, True))
    a = f(z, idx, top, rest=r)
    assert torch.equal(a, f(z, idx.int(), top.float(), rest=r))
    # views: classes and rows strided, an odd start address
    wide = torch.empty(12, 1403, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:1401:2] = z
    assert torch.equal(a, f(wide[:, 1:1401:2], idx, top, rest=r))
    flat = torch.empty(z.numel() + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = z.reshape(-1)
    v = flat[1:].view_as(z).requires_grad_()
    b = f(v, idx, top, rest=r)
    (g,) = torch.autograd.grad(b, v)
    zz = z.clone().requires_grad_()
    (g2,) = torch.autograd.grad(f(zz, idx, top, rest=r), zz)
    assert torch.equal(a, b) and torch.equal(g, g2)
    # a model's output layout, [B, V, H, W]
    m = TopKDistill(temperature=2.0)
    img = z.float().view(3, 4, 700).movedim(-1, 1).reshape(3, 700, 2, 2)
    ii, tt = (t.view(3, 4, 9).movedim(-1, 1).reshape(3, 9, 2, 2) for t in (idx, top))
    c = m(img, ii, tt, r.view(3, 2, 2))
    assert torch.equal(c, m(img, ii.int(), tt.float(), r.view(3, 2, 2)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c2 = m(img, ii, tt, r.view(3, 2, 2))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c, c2)
    d = f(z.float(), idx, top, rest=r, temperature=2.0)
    assert abs(float(c) - float(d)) <= 1e-5 * abs(float(d))
    with pytest.raises(_lib.AccError):
        f(z, idx[:, :0], top[:, :0])
    with pytest.raises(_lib.AccError):
        f(z, idx, top[:, :8])
    with pytest.raises(_lib.AccError):
        f(z, idx.short(), top)
    with pytest.raises(_lib.AccError):
        f(z, idx, top, rest=r[:3])
    with pytest.raises(_lib.AccError):
        f(z.half(), idx, top)
    with pytest.raises(_lib.AccError):
        f(z, idx, top, dim=0)
    with pytest.raises(ValueError):
        f(z, idx, top.float().requires_grad_())
    big = torch.zeros(2, 300, device="cuda")
    with pytest.raises(_lib.AccError):
        f(big, torch.zeros(2, 257, dtype=torch.int32, device="cuda"), torch.zeros(2, 257, device="cuda"))


@pytest.mark.gpu
def test_gradient_against_differences():
    z, idx, top, r = _make(3, 40, 5, torch.float32, True, spread=1.0)
    zd = z.cuda().requires_grad_()
    loss = _fn()(zd, idx.cuda(), top.cuda(), rest=r.cuda(), temperature=1.3)
    (g,) = torch.autograd.grad(loss, zd)
    v = torch.randn(z.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)

    def value(t):
        return float(_reference(z.double() + t * v, idx, top, r, 1.3)[0].mean())

    h = 1e-4
    want = (value(h) - value(-h)) / (2 * h)
    have = float((g.double().cpu() * v).sum())
    assert abs(have - want) <= 1e-6 * float((g.double().cpu() * v).abs().sum()) + 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,K", [(260, 2049, 9), (300, 33001, 5), (257, 70001, 64), (1030, 21, 3)])
def test_many_rows(R, V, K, dtype):
    """One block a row, each number of threads; the loss checked on every row, the gradient
    on rows spread over the batch (the 64-bit reference is a loop)."""
    z, idx, top, r = _make(R, V, 1, dtype, True)
    g = torch.Generator().manual_seed(5)
    idx = torch.randint(0, V, (R, K), generator=g)
    top = torch.randn(R, K, generator=g).to(dtype)
    idx[R // 2] = -1
    pick = [0, 1, R // 2, R - 2, R - 1]
    loss64, dz64, tl, td, live = _reference(z[pick], idx[pick], top[pick], r[pick], 1.7)
    zd = z.cuda().requires_grad_()
    args = (idx.cuda(), top.cuda())
    kw = dict(rest=r.cuda(), temperature=1.7)
    per = _fn()(zd, *args, reduction="none", **kw)
    _close(per[pick], loss64, tl, "loss")
    (dn,) = torch.autograd.grad(per, zd, torch.ones_like(per))
    _close(dn[pick], dz64, td, "dz none")
    n = R - 1
    mean = _fn()(zd, *args, **kw)
    want = per.detach().double().sum() / n
    assert abs(float(mean) - float(want)) <= 4 * U * abs(float(want))
    (dm,) = torch.autograd.grad(mean, zd)
    _close(dm[pick], dz64 / n, (td + 8 * U * dz64.abs()) / n, "dz mean")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "long", "planes"])
def test_held_gradient(layout):
    """The forward's gradient is handed out once; other upstream gradients, a second backward
    of the same graph and an accumulated leaf are right too."""
    f = _fn()
    R, V = {"rows": (24, 500), "long": (260, 5001), "planes": (24, 21)}[layout]
    z, idx, top, r = (t.cuda() for t in _make(R, V, 6, torch.float32, True))
    dim = -1
    if layout == "planes":
        z, idx, top = (t.view(2, R // 2, -1).movedim(-1, 1).contiguous() for t in (z, idx, top))
        r, dim = r.view(2, R // 2), 1

    def grad(up, **kw):
        zz = z.clone().requires_grad_()
        loss = f(zz, idx, top, rest=r, dim=dim, **kw)
        return torch.autograd.grad(loss, zz, torch.full_like(loss, up))[0]

    one = grad(1.0)
    for up in (0.5, -2.0, 4.0):  # powers of two: exact
        assert torch.equal(grad(up), one * up)
        assert torch.equal(grad(1.0, weight=up), one * up)
    assert torch.equal(grad(0.0), torch.zeros_like(one))
    zz = z.clone().requires_grad_()
    loss = f(zz, idx, top, rest=r, dim=dim)
    a = torch.autograd.grad(loss, zz, retain_graph=True)[0]
    b = torch.autograd.grad(loss, zz, torch.full_like(loss, 2.0), retain_graph=True)[0]
    c = torch.autograd.grad(loss, zz)[0]
    assert torch.equal(a, one) and torch.equal(b, 2 * one) and torch.equal(c, one)
    assert len({a.data_ptr(), b.data_ptr(), c.data_ptr()}) == 3
    zz = z.clone().requires_grad_()
    f(zz, idx, top, rest=r, dim=dim).backward()
    f(zz, idx, top, rest=r, dim=dim).backward()
    assert torch.equal(zz.grad, one + one)
    with torch.no_grad():
        v = f(z, idx, top, rest=r, dim=dim)
    assert torch.equal(v, loss.detach())


@pytest.mark.gpu
def test_backward_alone_captured():
    """The forward runs eagerly, its backward is captured and replayed with other upstream
    gradients: each replay writes what its upstream asks for."""
    f = _fn()
    z, idx, top, r = (t.cuda() for t in _make(24, 500, 6, torch.float32, True))
    want = {}
    for up in (1.0, 0.5, 2.0):
        zz = z.clone().requires_grad_()
        loss = f(zz, idx, top, rest=r)
        want[up] = torch.autograd.grad(loss, zz, torch.full_like(loss, up))[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        zz = z.clone().requires_grad_()
        loss = f(zz, idx, top, rest=r)
        up = torch.ones_like(loss)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            (dz,) = torch.autograd.grad(loss, zz, up)
            out = dz.clone()
            dz.add_(1.0)  # a consumer that works in place
    for u in (2.0, 1.0, 1.0, 0.5, 1.0):
        up.fill_(u)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[u]), u


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "long", "planes"])
def test_capture_and_repeatability(layout):
    f = _fn()
    V = {"rows": 500, "long": 9001, "planes": 21}[layout]
    z, idx, top, r = _make(24, V, 6, torch.float32, True)
    dim = -1
    args = [t.cuda() for t in (z, idx, top, r)]
    if layout == "planes":
        args[:3] = [t.view(2, 12, -1).movedim(-1, 1).contiguous() for t in args[:3]]
        args[3] = args[3].view(2, 12)
        dim = 1
    zd = args[0].requires_grad_()

    def step():
        loss = f(zd, args[1], args[2], rest=args[3], dim=dim)
        return [loss, *torch.autograd.grad(loss, zd)]

    eager = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
        again = step()
        torch.cuda.synchronize()
        for a, b, c in zip(eager, out, again):
            assert torch.equal(a, b) and torch.equal(a, c)
    with torch.no_grad():  # new inputs in the graph's buffers
        zd += torch.randn(zd.shape, generator=torch.Generator().manual_seed(3)).cuda()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(step(), out):
        assert torch.equal(a, b)
