"""The norms around a residual block (accunet/blocknorm.py) against the formulas in 64 bits.

Tolerance: with u = 2^-24, a statistic over C fp32 terms is a tree of at most
8 + 6 + 16 additions, so norm(v) is off by at most ~32 u * k, k = max|v| / std + max|norm(v)|
of the row; a gradient passes through both norms (k1 * k2) and at most four such steps:
128 * u * k1 * k2 * M, M the sum of the magnitudes that an element adds up. Parameter and
shared-gate gradients add at most P / (4 * blocks) + 16 such terms one after another, here
below 64. Stored bf16 adds half a step, eps / 2 of the value."""
import pytest
import torch

from accunet import _lib

U = 2.0 ** -24


def _mods():
    from accunet import blocknorm
    return blocknorm


# ---------------------------------------------------------------------- refusals (CPU)
def test_refusals_on_the_host():
    bn = _mods()
    x = torch.zeros(2, 3, 8)
    with pytest.raises(_lib.AccError):
        bn.sandwich_norm(x, x)  # host tensors
    with pytest.raises(ValueError):
        bn.norm(x, kind="batch")
    with pytest.raises(ValueError):
        bn.SandwichNorm(8, kind="batch")
    lib = _lib.load()
    ok = 16
    # f without r, a gate without f, a gate mode without a gate, rows no sample divides,
    # channels past the limit, an unknown storage type: refused before any launch
    f = lib.accunet_blocknorm_fwd
    assert f(ok, ok, None, None, None, None, 0, None, None, 1, 1e-5, None, ok, None, 4, 4, 8, 0, None) == -2
    assert f(ok, None, None, None, None, ok, 1, None, None, 1, 1e-5, None, ok, None, 4, 4, 8, 0, None) == -2
    assert f(ok, ok, None, None, None, None, 1, None, None, 1, 1e-5, ok, ok, None, 4, 4, 8, 0, None) == -2
    assert f(ok, ok, None, None, None, ok, 3, None, None, 1, 1e-5, ok, ok, None, 4, 4, 8, 0, None) == -2
    assert f(ok, ok, None, None, None, ok, 1, None, None, 1, 1e-5, ok, ok, None, 5, 4, 8, 0, None) == -1
    assert f(ok, ok, None, None, None, None, 0, None, None, 1, 1e-5, ok, ok, None, 4, 4, 8193, 0, None) == -1
    assert f(ok, ok, None, None, None, None, 0, None, None, 1, 1e-5, ok, ok, None, 0, 1, 8, 0, None) == -1
    assert f(ok, ok, None, None, None, None, 0, None, None, 1, 1e-5, ok, ok, None, 4, 4, 8, 2, None) == -2
    b = lib.accunet_blocknorm_bwd
    n = lib.accunet_blocknorm_ws_elems(4, 4, 8, 0)
    assert n > 0 and lib.accunet_blocknorm_ws_elems(4, 3, 8, 0) == 0
    assert b(ok, ok, None, None, None, None, 0, None, 1, ok, None, None, ok, ok, None, ok, ok, n,
             4, 4, 8, 0, None) == -2  # neither dr nor dh
    assert b(ok, ok, None, None, None, None, 0, None, 1, ok, ok, ok, ok, ok, None, ok, ok, n - 1,
             4, 4, 8, 0, None) == -2  # workspace too small


# ----------------------------------------------------------------------- the reference
def _norm64(v, kind, eps):
    d = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return d * rstd, rstd


def _inputs(B, L, C, dtype, gate, affine, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    def act(t):
        return t.to(dtype)

    d = {"x": act(2 * rn(B, L, C) + rn(C)), "f": act(rn(B, L, C) + 0.3),
         "dr": act(rn(B, L, C)), "dh": act(rn(B, L, C)),
         "g": None if gate == "none" else act(rn(B, 1, C) if gate == "sample" else rn(B, L, C))}
    for k, base in (("w1", 1.0), ("b1", 0.0), ("s", 0.6), ("w2", 1.0), ("b2", 0.0)):
        d[k] = (base + 0.3 * rn(C)).float() if affine else None
    return d


LEAVES = ("x", "f", "w1", "b1", "s", "g", "w2", "b2")


def _reference(d, kind, eps, use_r=True, use_h=True):
    """Outputs, gradients and, for each, the bound of the module docstring."""
    C = d["x"].shape[-1]
    one, zero = torch.ones(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)
    w = {k: (d[k].double() if d[k] is not None else v) for k, v in
         (("w1", one), ("b1", zero), ("s", one), ("w2", one), ("b2", zero))}
    x, f = d["x"].double(), d["f"].double()
    g = d["g"].double() if d["g"] is not None else torch.ones_like(x[:, :1])
    fh, r1 = _norm64(f, kind, eps)
    u = fh * w["w1"] + w["b1"]
    r = x + w["s"] * g * u
    rh, r2 = _norm64(r, kind, eps)
    h = rh * w["w2"] + w["b2"]

    def kappa(v, vh, rs):
        return (v.abs().amax(-1, keepdim=True) * rs + vh.abs().amax(-1, keepdim=True))

    k1, k2 = kappa(f, fh, r1), kappa(r, rh, r2)
    aw1, asg = w["w1"].abs(), (w["s"] * g).abs()
    mu = (fh.abs() + k1) * aw1 + w["b1"].abs()
    mr = x.abs() + asg * mu
    # the error of r reaches rhat over the row's largest magnitude
    k2 = k2 + mr.amax(-1, keepdim=True) * r2
    mh = (rh.abs() + k2) * w["w2"].abs() + w["b2"].abs()
    dr = d["dr"].double() if use_r else torch.zeros_like(x)
    dh = d["dh"].double() if use_h else torch.zeros_like(x)

    def nb(e, vh, rs):
        m = e - vh * (e * vh).mean(-1, keepdim=True)
        if kind == "layer":
            m = m - e.mean(-1, keepdim=True)
        return m * rs

    def nbmag(e, vh, rs):
        return rs * (e + e.mean(-1, keepdim=True) + (vh.abs() + 1) * (e * (vh.abs() + 1)).mean(-1, keepdim=True))

    gr = dr + nb(dh * w["w2"], rh, r2)
    mgr = dr.abs() + nbmag((dh * w["w2"]).abs(), rh, r2) * k2
    du = gr * w["s"] * g
    mdu = mgr * asg
    df = nb(du * w["w1"], fh, r1)
    mdf = nbmag(mdu * aw1, fh, r1) * k1
    ax = (0, 1)
    full = lambda t: t.expand_as(x)  # noqa: E731
    val = {"r": r, "h": h, "x": gr, "f": df, "w1": (du * fh).sum(ax), "b1": du.sum(ax),
           "s": (gr * g * u).sum(ax), "w2": (dh * rh).sum(ax), "b2": dh.sum(ax),
           "g": full(gr * w["s"] * u)}
    mag = {"r": mr, "h": mh, "x": mgr, "f": mdf, "w1": (mdu * (fh.abs() + k1)).sum(ax),
           "b1": mdu.sum(ax), "s": (mgr * g.abs() * mu).sum(ax),
           "w2": (dh.abs() * (rh.abs() + k2)).sum(ax), "b2": dh.abs().sum(ax),
           "g": full(mgr * w["s"].abs() * mu)}
    if d["g"] is not None and d["g"].shape[1] == 1 and x.shape[1] != 1:
        val["g"], mag["g"] = val["g"].sum(1, keepdim=True), mag["g"].sum(1, keepdim=True)
    return val, {k: 128 * U * m for k, m in mag.items()}


def _compare(name, got, want, tol):
    got = got.detach().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if got.dtype == torch.bfloat16:
        tol = tol + want.abs() * torch.finfo(torch.bfloat16).eps / 2 * (1 + 2 ** -8)
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0, (name, float(over.max()), float((got.double() - want).abs().max()))


def _run(d, kind, eps=1e-5, use_r=True, use_h=True):
    bn = _mods()
    dev = {k: (v.cuda() if v is not None else None) for k, v in d.items()}
    for k in LEAVES:
        if dev[k] is not None:
            dev[k].requires_grad_()
    r, h = bn.sandwich_norm(dev["x"], dev["f"], dev["w1"], dev["b1"], dev["s"], dev["g"],
                            dev["w2"], dev["b2"], kind=kind, eps=eps)
    outs = [o for o, u in ((r, use_r), (h, use_h)) if u]
    grads = [dev[k] for k, u in (("dr", use_r), ("dh", use_h)) if u]
    leaves = [k for k in LEAVES if dev[k] is not None]
    gs = torch.autograd.grad(outs, [dev[k] for k in leaves], grads, allow_unused=True)
    return r, h, dict(zip(leaves, gs))


SHAPES = [(1, 1, 1), (2, 1, 8), (3, 5, 33), (2, 70, 160), (5, 9, 256), (2, 17, 260), (1, 37, 512),
          (2, 6, 777), (3, 4, 1024), (1, 5, 2047), (1, 6, 4096), (1, 3, 8192), (1, 2, 8191),
          (1100, 3, 16), (2, 2500, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sandwich_norm_matches_64_bits(shape, dtype):
    for i, (kind, gate, affine) in enumerate((("layer", "sample", True), ("rms", "element", True),
                                              ("layer", "none", False), ("rms", "sample", False))):
        # a layer norm over one channel is zero whatever the input: only rms is comparable
        if shape[-1] == 1 and kind == "layer":
            continue
        d = _inputs(*shape, dtype, gate, affine, seed=i)
        r, h, got = _run(d, kind)
        val, tol = _reference(d, kind, 1e-5)
        _compare("r", r, val["r"], tol["r"])
        _compare("h", h, val["h"], tol["h"])
        for k, t in got.items():
            _compare(k, t, val[k], tol[k])


@pytest.mark.gpu
@pytest.mark.parametrize("use_r,use_h", [(True, False), (False, True)])
def test_one_output_used(use_r, use_h):
    d = _inputs(2, 9, 96, torch.float32, "sample", True)
    _, _, got = _run(d, "layer", use_r=use_r, use_h=use_h)
    val, tol = _reference(d, "layer", 1e-5, use_r, use_h)
    for k, t in got.items():
        if t is not None:
            _compare(k, t, val[k], tol[k])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_alone_and_block_without_a_next_norm(kind):
    bn = _mods()
    d = _inputs(2, 11, 320, torch.float32, "none", True)
    x, w2, b2 = (d[k].cuda().requires_grad_() for k in ("x", "w2", "b2"))
    h = bn.norm(x, w2, b2, kind=kind)
    gx, gw, gb = torch.autograd.grad(h, [x, w2, b2], d["dh"].cuda())
    z = dict(d, f=torch.zeros_like(d["f"]), w1=None, b1=None, s=None)
    val, tol = _reference(z, kind, 1e-5, use_r=False)
    for k, t in (("h", h), ("x", gx), ("w2", gw), ("b2", gb)):
        _compare(k, t, val[k], tol[k])
    # pre=False: r alone
    m = bn.SandwichNorm(320, kind=kind, scale_init=0.5, pre=False).cuda()
    r, none = m(d["x"].cuda(), d["f"].cuda())
    assert none is None
    e = dict(d, w1=None, b1=None, s=torch.full((320,), 0.5), w2=None, b2=None)
    val, tol = _reference(e, kind, 1e-5)
    _compare("r", r, val["r"], tol["r"])
    r.sum().backward()
    assert m.scale.grad is not None and m.post_weight.grad is not None and m.post_bias.grad is not None


@pytest.mark.gpu
def test_gradients_against_differences():
    """d(sum(r*dr + h*dh)) along a random direction of every leaf, against a central
    difference of the 64-bit forward."""
    d = _inputs(2, 5, 24, torch.float32, "sample", True)
    _, _, got = _run(d, "layer")
    gen = torch.Generator().manual_seed(5)
    for k in LEAVES:
        v = torch.randn(d[k].shape, generator=gen, dtype=torch.float64)

        def value(t):
            e = dict(d)
            e[k] = d[k].double() + t * v
            val, _ = _reference(e, "layer", 1e-5)
            return float((val["r"] * d["dr"].double()).sum() + (val["h"] * d["dh"].double()).sum())

        step = 1e-4
        want = (value(step) - value(-step)) / (2 * step)
        have = float((got[k].double().cpu() * v).sum())
        mag = float((got[k].double().cpu() * v).abs().sum())
        # the difference's own truncation is step^2 of a third derivative of order 10
        assert abs(have - want) <= 2e-6 * mag + 1e-5, (k, have, want)


@pytest.mark.gpu
def test_strides_empty_rows_and_refusals():
    bn = _mods()
    base = torch.randn(4, 6, 64, device="cuda")
    x = base.transpose(0, 1)[:, :, 1:42]  # neither contiguous nor 16-byte aligned
    f = torch.randn(6, 4, 41, device="cuda")
    r, h = bn.sandwich_norm(x, f)
    r2, h2 = bn.sandwich_norm(x.contiguous(), f)
    assert torch.equal(r, r2) and torch.equal(h, h2)
    # an aligned row length at an unaligned address (a view one element in): its sums run
    # over single elements, in another order than over 16 bytes, so bits may differ and the
    # bound of the module docstring holds for both
    flat = torch.randn(3 * 64 + 1, device="cuda")
    y = flat[1:].view(3, 64)
    y64 = y.double().cpu()
    want, rstd = _norm64(y64, "layer", 1e-5)
    kappa = y64.abs().amax(-1, keepdim=True) * rstd + want.abs().amax(-1, keepdim=True)
    for t in (y, y.clone()):
        _compare("h", bn.norm(t), want, 128 * U * (want.abs() + kappa))
    # one row without a batch axis; another stream
    assert torch.equal(bn.norm(f[0, 0]), bn.norm(f)[0, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r3, h3 = bn.sandwich_norm(x, f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(r, r3) and torch.equal(h, h3)
    # constant rows: zero variance
    c = torch.full((2, 48), 3.0, device="cuda", requires_grad=True)
    hc = bn.norm(c)
    assert torch.equal(hc, torch.zeros_like(hc))
    # no rows
    e = torch.empty(2, 0, 16, device="cuda", requires_grad=True)
    g = torch.ones(2, 1, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    r, h = bn.sandwich_norm(e, e.detach(), w, gate=g)
    (r.sum() + h.sum()).backward()
    assert e.grad.shape == e.shape and torch.equal(w.grad, torch.zeros_like(w))
    assert torch.equal(g.grad, torch.zeros_like(g))
    with pytest.raises(_lib.AccError):
        bn.sandwich_norm(f, f, gate=torch.ones(6, 2, 41, device="cuda"))
    with pytest.raises(_lib.AccError):
        bn.sandwich_norm(f, f.bfloat16())
    with pytest.raises(_lib.AccError):
        bn.sandwich_norm(f, f[:, :2])
    with pytest.raises(_lib.AccError):
        bn.norm(f, torch.ones(41, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(_lib.AccError):
        bn.norm(f, torch.ones(40, device="cuda"))
    with pytest.raises(_lib.AccError):
        bn.norm(torch.zeros(1, 8193, device="cuda"))
    with pytest.raises(_lib.AccError):
        bn.norm(f.half())
    with pytest.raises(ValueError):
        bn.sandwich_norm(f, f, pre=False, pre_weight=torch.ones(41, device="cuda"))


@pytest.mark.gpu
def test_capture_streams_and_repeatability():
    bn = _mods()
    d = {k: (v.cuda() if v is not None else None)
         for k, v in _inputs(3, 200, 160, torch.bfloat16, "sample", True).items()}
    for k in LEAVES:
        d[k].requires_grad_()
    leaves = [d[k] for k in LEAVES]

    def step():
        r, h = bn.sandwich_norm(d["x"], d["f"], d["w1"], d["b1"], d["s"], d["g"], d["w2"], d["b2"])
        return [r, h, *torch.autograd.grad([r, h], leaves, [d["dr"], d["dh"]])]

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
        again = step()  # eager work between the replays
        torch.cuda.synchronize()
        for a, b, c in zip(eager, out, again):
            assert torch.equal(a, b) and torch.equal(a, c)
