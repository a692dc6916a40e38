"""The token-block operators together, as a training step uses them: norm -> 8-bit linear ->
GELU -> 8-bit linear -> norm, scale and gate with the residual add and the next norm -> 8-bit
head -> distillation from a teacher's top logits; and the UNeXt options that call them.

Each stage of the run is held, forward and backward, to its own 64-bit reference on the
inputs and output gradients that it had in the run (a quantised value near a rounding border
may fall on either side for inputs one fp32 rounding apart, so the chain as a whole has no
64-bit value to compare with). Tolerances: those of the operators' own tests."""
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import test_blocknorm as TN  # noqa: E402
import test_distill as TD  # noqa: E402
import test_fp8 as TF  # noqa: E402


def test_default_unext_is_the_reference_network():
    from accunet.unext import UNext
    base, opt = UNext(3, 1).state_dict(), UNext(3, 1, linear="fp8").state_dict()
    assert list(base) == list(opt)
    extra = set(UNext(3, 1, sandwich=True).state_dict()) - set(base)
    assert {k.split(".", 2)[2] for k in extra} == {"post_norm.weight", "post_norm.bias", "scale"}
    with pytest.raises(ValueError):
        UNext(3, 1, linear="int8")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_stage_by_stage(dtype):
    from accunet import blocknorm, fp8
    from accunet.loss import TopKDistill
    B, L, C, H, V, K = 3, 65, 160, 200, 333, 7
    gen = torch.Generator().manual_seed(1)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    par = {"w1": rn(H, C) / C ** .5, "b1": .1 * rn(H), "w2": rn(C, H) / H ** .5, "b2": .1 * rn(C),
           "wh": rn(V, C) / C ** .5, "n1": 1 + .1 * rn(C), "pw": 1 + .1 * rn(C), "pb": .1 * rn(C),
           "sc": .5 + .1 * rn(C), "qw": 1 + .1 * rn(C), "qb": .1 * rn(C)}
    par = {k: v.cuda().requires_grad_() for k, v in par.items()}
    x = rn(B, L, C).to(dtype).cuda().requires_grad_()
    gate = rn(B, 1, C).to(dtype).cuda().requires_grad_()
    idx = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(B * L)]).view(B, L, K)
    top, rest = 2 * rn(B, L, K), torch.rand(B, L, generator=gen) * .5

    h0 = blocknorm.norm(x, par["n1"], kind="rms")
    y1 = fp8.linear(h0, par["w1"], par["b1"])
    a1 = torch.nn.functional.gelu(y1)
    f = fp8.linear(a1, par["w2"], par["b2"])
    r, h = blocknorm.sandwich_norm(x, f, par["pw"], par["pb"], par["sc"], gate, par["qw"], par["qb"])
    z = fp8.linear(h, par["wh"])
    mid = (h0, y1, a1, f, r, h, z)
    for t in mid:
        t.retain_grad()
    loss = TopKDistill(temperature=2.0, dim=-1)(z, idx.cuda(), top.cuda(), rest.cuda())
    (loss + 0.25 * r.float().square().mean()).backward()  # r is the next block's residual too
    c = {n: t.detach().cpu() for n, t in zip(("h0", "y1", "a1", "f", "r", "h", "z"), mid)}
    g = {n: t.grad.cpu() for n, t in zip(("h0", "y1", "a1", "f", "r", "h", "z"), mid)}
    p = {k: v.detach().cpu() for k, v in par.items()}

    def linear(inp, w, b, out, dout, gin, gw, gb):
        a, d = inp.reshape(-1, inp.shape[-1]), dout.reshape(-1, dout.shape[-1])
        wg = TF._grid(w, 128)[0]
        TF._product_ok(out.reshape(-1, out.shape[-1]), TF._grid(a)[0], wg, b)
        TF._product_ok(gin.reshape(a.shape), TF._grid(d)[0], wg.t().contiguous())
        TF._product_ok(gw, TF._grid(d.t().contiguous())[0], TF._grid(a.t().contiguous())[0])
        if gb is not None:
            want, mag = d.double().sum(0), d.double().abs().sum(0)
            assert bool(((gb.double().cpu() - want).abs() <= 32 * TF.U * mag).all())

    linear(c["h0"], p["w1"], p["b1"], c["y1"], g["y1"], g["h0"], par["w1"].grad, par["b1"].grad)
    linear(c["a1"], p["w2"], p["b2"], c["f"], g["f"], g["a1"], par["w2"].grad, par["b2"].grad)
    linear(c["h"], p["wh"], None, c["z"], g["z"], g["h"], par["wh"].grad, None)
    d = {"x": x.detach().cpu(), "f": c["f"], "dr": g["r"], "dh": g["h"], "g": gate.detach().cpu(),
         "w1": p["pw"], "b1": p["pb"], "s": p["sc"], "w2": p["qw"], "b2": p["qb"]}
    val, tol = TN._reference(d, "layer", 1e-5)
    for k, t in (("r", r), ("h", h), ("f", g["f"]), ("g", gate.grad), ("w1", par["pw"].grad),
                 ("b1", par["pb"].grad), ("s", par["sc"].grad), ("w2", par["qw"].grad),
                 ("b2", par["qb"].grad)):
        TN._compare(k, t, val[k], tol[k])
    l64, dz64, tl, td, live = TD._reference(c["z"].reshape(-1, V), idx.view(-1, K),
                                            top.view(-1, K), rest.view(-1), 2.0)
    n = B * L
    TD._close(loss, l64.sum() / n, tl.sum() / n + 8 * TD.U * l64.sum() / n, "loss")
    TD._close(g["z"].reshape(-1, V), dz64 / n, (td + 8 * TD.U * dz64.abs()) / n, "dz")
    # x: the residual branch's gradient plus the first norm's, added by autograd in x's type
    zero = dict(d, f=torch.zeros_like(d["f"]), w1=None, b1=None, s=None, g=None, w2=p["n1"],
                b2=None, dh=g["h0"])
    v2, t2 = TN._reference(zero, "rms", 1e-5, use_r=False)
    TN._compare("h0", h0, v2["h"], t2["h"])
    want = val["x"] + v2["x"]
    bound = tol["x"] + t2["x"] + (torch.finfo(dtype).eps / 2 * (val["x"].abs() + v2["x"].abs()) * 1.01)
    TN._compare("x", x.grad, want, bound + torch.finfo(dtype).eps / 2 * want.abs())


@pytest.mark.gpu
def test_unext_options_train():
    """UNext(sandwich=True): output and every gradient against the same network with the
    fused norm replaced by torch's operations, within four times what one fp32 rounding of
    the input changes (eval-mode statistics); UNext(linear="fp8", sandwich=True) with the
    distillation loss: finite gradients for every parameter, repeatable bit for bit."""
    import torch.nn.functional as F
    from accunet import unext
    from accunet.loss import TopKDistill
    torch.manual_seed(0)
    m = unext.UNext(3, 6, sandwich=True).cuda().eval()
    x = torch.randn(2, 3, 64, 64, device="cuda")
    dy = torch.randn(2, 6, 64, 64, device="cuda")
    names = [n for n, _ in m.named_parameters()]
    params = [q for _, q in m.named_parameters()]

    def step(inp):
        y = m(inp)
        return [y.detach(), *torch.autograd.grad(y, params, dy)]

    def plain(x, f, w1, b1, s, g, w2, b2, eps=1e-5):
        C = (x.shape[-1],)
        r = x + s * F.layer_norm(f, C, w1, b1, eps)
        return r, F.layer_norm(r, C, w2, b2, eps)

    got = step(x)
    fused = unext.sandwich_norm
    try:
        unext.sandwich_norm = plain
        want = step(x)
        moved = [step(x * (1 + e)) for e in (2.0 ** -23, -(2.0 ** -23))]
    finally:
        unext.sandwich_norm = fused
    for i, n in enumerate(["y"] + names):
        noise = max(float((mv[i] - want[i]).norm()) for mv in moved)
        scale = float(want[i].norm())
        assert float((got[i] - want[i]).norm()) <= 4 * noise + 1e-5 * scale + 1e-12, n

    m = unext.UNext(3, 6, sandwich=True, linear="fp8").cuda().train()
    params = list(m.parameters())
    crit = TopKDistill(temperature=2.0)
    idx = torch.stack([torch.randperm(6)[:3] for _ in range(2 * 64 * 64)]).view(2, 64, 64, 3)
    idx = idx.movedim(-1, 1).contiguous().cuda()
    top = torch.randn(2, 3, 64, 64, device="cuda")
    rest = torch.rand(2, 64, 64, device="cuda") * .3
    out = []
    for _ in range(2):
        loss = crit(m(x), idx, top, rest)
        out.append([loss.detach(), *torch.autograd.grad(loss, params)])
    for a, b in zip(*out):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
    grads = dict(zip(names, out[0][1:]))
    for n in ("block1.0.mlp.fc1.weight", "block2.0.scale", "dblock1.0.post_norm.weight"):
        assert float(grads[n].abs().max()) > 0, n


@pytest.mark.gpu
def test_unext_options_in_a_captured_step():
    """TrainStep's graph mode with the options on: three replayed steps give the eager
    steps' losses and parameters bit for bit."""
    from accunet.train import TrainStep
    from accunet.unext import UNext
    gen = torch.Generator().manual_seed(3)
    xs = [torch.randn(2, 3, 64, 64, generator=gen).cuda() for _ in range(3)]
    ys = [(torch.rand(2, 1, 64, 64, generator=gen) < 0.4).float().cuda() for _ in range(3)]
    torch.manual_seed(0)
    state = UNext(3, 1, sandwich=True, linear="fp8").state_dict()
    runs = []
    for graph in (True, False):
        m = UNext(3, 1, sandwich=True, linear="fp8")
        m.load_state_dict(state)
        step = TrainStep(m.cuda().train(), lr=1e-3, graph=graph)
        losses = [float(step(x, y)) for x, y in zip(xs, ys)]
        runs.append((losses, [p.detach().clone() for p in m.parameters()]))
        del step, m
    assert runs[0][0] == runs[1][0]
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


def _near(big, small):
    """Two calls on the same rows: one bf16 step apart at most, 2^-13 of the largest value on
    top for fp32 sums in another order (up to 2^11 terms, 2^-24 each)."""
    a, b = big.detach().double(), small.detach().double()
    bound = torch.finfo(torch.bfloat16).eps * b.abs() + 2.0 ** -13 * float(b.abs().max())
    assert float(b.abs().max()) > 0 and bool(((a - b).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "rows", "planes", "linear"])
def test_offsets_past_32_bits(op):
    """More than 2^31 elements: the last rows are what a call on these rows alone gives."""
    from accunet import blocknorm, distill, fp8
    g = torch.Generator(device="cuda").manual_seed(3)

    def rand(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)

    n = 300

    def leaf(t):
        return t.detach().clone().requires_grad_()

    if op == "norm":
        P, C = 2 ** 22 + 3, 520
        x, f = rand(P, C).requires_grad_(), rand(P, C).requires_grad_()
        r, h = blocknorm.sandwich_norm(x, f)
        torch.autograd.backward([r, h], [x.detach(), f.detach()])
        xs, fs = leaf(x[-n:]), leaf(f[-n:])
        rs, hs = blocknorm.sandwich_norm(xs, fs)
        torch.autograd.backward([rs, hs], [xs.detach(), fs.detach()])
        for a, b in ((r, rs), (h, hs), (x.grad, xs.grad), (f.grad, fs.grad)):
            _near(a[-n:], b)
    elif op == "linear":
        M, K, N = 2 ** 21 + 300, 1040, 8
        x = rand(M, K).requires_grad_()
        w = torch.randn(N, K, generator=g, device="cuda", requires_grad=True)
        first = (M - n) // 128 * 128  # the first of a block of 128 tokens
        dy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
        dy[first:].normal_(generator=g)
        y = fp8.linear(x, w)
        y.backward(dy)
        xs, ws = leaf(x[first:]), leaf(w)
        ys = fp8.linear(xs, ws)
        ys.backward(dy[first:])
        for a, b in ((y[first:], ys), (x.grad[first:], xs.grad), (w.grad, ws.grad)):
            _near(a, b)
        assert not x.grad[:first].any()
    else:
        shape, dim = ((2 ** 21 + 70001, 1001), -1) if op == "rows" else ((4, 21, 2 ** 25 + 5), 1)
        K = [s if i != dim % len(shape) else 2 for i, s in enumerate(shape)]
        z = rand(*shape).requires_grad_()
        V = shape[dim]
        idx = torch.randint(0, V, K, generator=g, device="cuda", dtype=torch.int32)
        top = rand(*K)
        loss = distill.topk_distill(z, idx, top, reduction="none", dim=dim)
        loss.backward(torch.ones_like(loss))
        cut = (slice(-n, None),) if op == "rows" else (slice(3, 4), slice(None), slice(-n, None))
        zs = leaf(z[cut])
        ls = distill.topk_distill(zs, idx[cut], top[cut], reduction="none", dim=dim)
        ls.backward(torch.ones_like(ls))
        _near(loss[-n:] if op == "rows" else loss[3:, -n:], ls)
        _near(z.grad[cut], zs.grad)
