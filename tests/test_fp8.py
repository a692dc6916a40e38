"""The 8-bit linear layer (accunet/fp8.py): quantised values bit for bit against their
definition in 64 bits, products against the 64-bit product of those values.

Tolerance of a product: every factor is exact, so only the sum over the contracted axis
rounds. With u = 2^-24, n terms added one after another are off by at most n * u * sum |a b|
to first order; 32 or 128 terms are one instruction (counted as if added in turn) and the
instructions follow each other, so n <= 128 + K / 32. For bf16 outputs the instruction
keeps, of 8 products, 13 bits below the largest: at most 7 * 2^-13 of it a group, bounded by
the product of the group's largest factors; the store adds half a step, eps / 2 of the value."""
import math

import pytest
import torch

from accunet import _lib, kern

U = 2.0 ** -24


def _mod():
    from accunet import fp8
    return fp8


# ---------------------------------------------------------------------- refusals (CPU)
def test_refusals_on_the_host():
    fp8 = _mod()
    with pytest.raises(_lib.AccError):
        fp8.quantize(torch.zeros(2, 8))
    with pytest.raises(_lib.AccError):
        fp8.linear(torch.zeros(2, 8), torch.zeros(4, 8))
    q, s = torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.full((4, 4), 127, dtype=torch.uint8)
    assert fp8.Fp8Blocks(q, s, 4, 77, True).shape == (4, 77)
    for bad in ((q[:3], s, 4, 77), (q, s[:, :3], 4, 77), (q, s, 4, 129), (q.float(), s, 4, 77),
                (q.t(), s, 128, 4), (s, q, 4, 77)):
        with pytest.raises(_lib.AccError):
            fp8.Fp8Blocks(*bad, True)
    lib = _lib.load()
    ok = 16
    q = lib.accunet_fp8_quantize
    assert q(ok, 0, ok, ok, None, None, 0, 8, 0, None) == -1
    assert q(ok, 0, ok, None, None, None, 2, 8, 0, None) == -2   # q without s
    assert q(ok, 0, ok, ok, ok, None, 2, 8, 0, None) == -2       # qt without st
    assert q(ok, 0, ok, ok, None, None, 2, 8, 3, None) == -2     # storage type
    assert q(ok, 0, ok, ok, None, None, 2, (1 << 22) + 1, 0, None) == -1
    fwd, bwd, al = lib.accunet_fp8_linear_fwd, lib.accunet_fp8_linear_bwd, 256
    n = lib.accunet_fp8_linear_ws_bytes(8, 8, 4096, 1)
    k = lib.accunet_fp8_linear_save_bytes(8, 8, 4096, 1, 1)
    assert n > 0 and k > 0 and lib.accunet_fp8_linear_ws_bytes(0, 8, 8, 1) == 0

    def f_(x=ok, w=ok, wq=None, wqs=None, need_w=1, need_wt=1, save=al, kb=k, ws=al, nb=n, M=8, dt=0):
        return fwd(x, w, wq, wqs, None, ok, need_w, need_wt, save, kb, ws, nb, M, 8, 4096, dt, None)

    assert f_(M=0) == -1 and f_(dt=2) == -2 and f_(x=None) == -2 and f_(nb=n - 1) == -2
    assert f_(kb=k - 1) == -2 and f_(save=None) == -2 and f_(ws=16) == -2 and f_(wq=ok) == -2
    assert f_(w=None) == -2 and f_(w=None, wq=ok, wqs=ok) == -2  # need_wt without w
    assert f_(w=None, wq=8, wqs=ok, need_wt=0) == -2             # alignment
    m = lib.accunet_fp8_linear_bwd_ws_bytes(8, 8, 4096, 1, 1, 1)

    def b_(dy=ok, save=al, need_w=1, need_wt=1, dx=ok, dw=ok, db=ok, mb=m):
        return bwd(dy, save, need_w, need_wt, None, None, dx, dw, db, al, mb, 8, 8, 4096, 0, None)

    assert b_(dy=None) == -2 and b_(mb=m - 1) == -2 and b_(save=None) == -2
    assert b_(dx=None, dw=None, db=None) == -2 and b_(need_w=0) == -2 and b_(need_wt=0) == -2


# ----------------------------------------------------------------------- the reference
def _two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(v):
    """v (|v| <= 448) to nearest even e4m3."""
    _, k = torch.frexp(v)
    ulp = _two((k - 1).clamp(min=-6) - 3)
    return torch.round(v / ulp) * ulp


def _grid(x, rows=1):
    """Values of x [R, C] on the scales of its blocks of rows x 128, in 64 bits, and the
    biased exponents [R, blocks]."""
    x = x.double()
    R, C = x.shape
    out, byte = torch.empty_like(x), torch.empty(R, -(-C // 128), dtype=torch.int64)
    for i in range(0, R, rows):
        for j in range(0, C, 128):
            b = x[i:i + rows, j:j + 128]
            fin = torch.isfinite(b)
            a = float(torch.where(fin, b.abs(), torch.zeros_like(b)).max())
            e = 0 if a == 0 else max(-126, min(120, math.ceil(math.log2(a / 448.0))))
            while a > 448.0 * 2.0 ** e and e < 120:  # log2 next to an integer
                e += 1
            while a != 0 and e > -126 and a <= 448.0 * 2.0 ** (e - 1):
                e -= 1
            v = _round_e4m3(torch.where(fin, b, torch.zeros_like(b)) * 2.0 ** -e) * 2.0 ** e
            out[i:i + rows, j:j + 128] = torch.where(fin, v, torch.full_like(v, math.nan))
            byte[i:i + rows, j // 128] = e + 127
    return out, byte


def _data(R, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g) * torch.exp(1.5 * torch.randn(1, C, generator=g))
    return x.to(dtype)


def _assert_blocks(b, x, rows):
    want, byte = _grid(x.cpu(), rows)
    # values() is float32: the largest fp32 rounds up to 256 * 2^120 = 2^128, its infinity
    want = want.float().double()
    got = b.values().double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert bool(same.all()), int((~same).sum())
    n = byte.shape[1]
    assert torch.equal(b.s[:, :n].long().cpu(), byte)
    # padding: zeros behind the columns, 2^0 behind the scales
    assert not b.q.view(torch.uint8)[:, x.shape[1]:].any()
    assert bool((b.s[:, n:] == 127).all())


SIZES = [(1, 1), (1, 128), (3, 129), (128, 128), (130, 77), (257, 300), (5, 513), (64, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,C", SIZES)
def test_quantize(R, C, dtype):
    fp8 = _mod()
    x = _data(R, C, dtype).cuda()
    _assert_blocks(fp8.quantize(x), x, 1)
    b = fp8.quantize(x, square=True, transposed=True)
    _assert_blocks(b, x, 128)
    assert torch.equal(b.values().t().contiguous(), b.t.values())
    # the transposed form with blocks along the rows
    qt, st = fp8._new(C, R, x.device)
    q, sc = fp8._new(R, C, x.device)
    kern.fp8_quantize(x, False, q, sc, qt, st, R, C)
    _assert_blocks(fp8.Fp8Blocks(q, sc, R, C, False), x, 1)
    _assert_blocks(fp8.Fp8Blocks(qt, st, C, R, False), x.t().contiguous(), 1)


@pytest.mark.gpu
def test_values_of_every_scale():
    fp8 = _mod()
    x = torch.ldexp(torch.ones(246, 1), torch.arange(246).view(-1, 1) - 126 + 8) * 1.75
    b = fp8.quantize(x.cuda())
    assert torch.equal(b.s[:, 0].int().cpu(), torch.arange(1, 247, dtype=torch.int32))
    assert torch.equal(b.values().cpu(), x) and bool((b.q[:, 0].float() == 448).all())


@pytest.mark.gpu
def test_quantize_more_rows_than_a_launch_holds():
    """2^26 rows of one block take 2^32 threads: the rows on both sides of a cut, and the
    first and last, are what a call on these rows alone gives."""
    fp8 = _mod()
    R, C = 2 ** 26 + 3, 3
    x = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
    x.view(torch.int16).copy_(torch.arange(R * C, device="cuda").view(R, C) * 77 % 16256)
    b = fp8.quantize(x)
    for r in (0, 2 ** 25 - 40, 2 ** 26 - 77):
        part = fp8.quantize(x[r:r + 80])
        n = part.rows
        assert torch.equal(b.q[r:r + n].view(torch.uint8), part.q.view(torch.uint8))
        assert torch.equal(b.s[r:r + n], part.s)
        _assert_blocks(part, x[r:r + n], 1)


@pytest.mark.gpu
def test_quantize_values_at_the_edges():
    """Ties, the largest value and its neighbours, subnormals of e4m3 and of fp32, zeros,
    infinities and NaN, the largest and smallest fp32 scales."""
    fp8 = _mod()
    x = torch.zeros(16, 128)
    base = torch.arange(0, 128).float()
    x[0] = base * 3.5 + 0.0625
    x[1] = torch.linspace(-448, 448, 128)
    x[2, 0], x[2, 1:] = 448.0, torch.linspace(0, 2 ** -5, 127)
    x[3, 0] = torch.nextafter(torch.tensor(448.0), torch.tensor(500.0))
    x[3, 1:] = torch.linspace(1, 447, 127)
    x[4] = 1e-42 * base
    x[5] = 3e38 * torch.linspace(-1, 1, 128)
    x[6, 5], x[6, 7], x[6, 9], x[6, 11] = math.inf, -math.inf, math.nan, 2.0
    x[7] = math.inf
    x[8] = 2.0 ** -149
    x[9] = -0.0
    x[10] = torch.finfo(torch.float32).max
    x[11, 3] = torch.finfo(torch.float32).tiny
    x[12] = (base - 64) * 2.0 ** -9 + 2.0 ** -10
    x[12, 0] = 256.0
    x[13] = torch.where(base % 2 == 0, 17.0 * 2 ** 3, 19.0 * 2 ** 3)  # ties between steps of 16
    x[13, 0] = 448.0
    b = fp8.quantize(x.cuda())
    _assert_blocks(b, x.cuda(), 1)
    _assert_blocks(fp8.quantize(x.cuda(), square=True), x.cuda(), 128)


def _product_ok(got, a, b, bias=None):
    a, b = a.cuda(), b.cuda()  # fp64 products of fp64 values
    bias = bias.cuda() if bias is not None else None
    want = a @ b.t()
    mag = a.abs() @ b.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    K = a.shape[1]
    tol = (128 + K / 32 + 2) * U * mag
    got = got.detach().cuda()
    assert got.shape == want.shape
    if got.dtype == torch.bfloat16:
        top = [torch.nn.functional.pad(t.abs(), (0, -K % 8)).view(t.shape[0], -1, 8).amax(2)
               for t in (a, b)]
        tol = tol + 7 * 2.0 ** -13 * (top[0] @ top[1].t()) + want.abs() * torch.finfo(torch.bfloat16).eps / 2 * (1 + 2 ** -8)
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0, float(over.max())


GEMMS = [(1, 1, 1), (16, 40, 1100), (9, 250, 9000), (3000, 5700, 300), (1, 4096, 96), (1, 300, 513), (5, 17, 128), (17, 129, 1000), (64, 96, 2049), (128, 128, 512),
         (130, 250, 640), (333, 777, 160), (2, 640, 4100), (1000, 131, 257), (129, 1500, 96),
         (2500, 1400, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_linear_forward_and_gradients(M, N, K, dtype):
    fp8 = _mod()
    x, w = _data(M, K, dtype, 1).cuda(), _data(N, K, torch.float32, 2).cuda()
    b = _data(1, N, torch.float32, 3)[0].cuda()
    dy = _data(M, N, dtype, 4).cuda()
    for t in (x, w, b):
        t.requires_grad_()
    y = fp8.linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
    xc, wc, dyc = x.detach().cpu(), w.detach().cpu(), dy.cpu()
    wg = _grid(wc, 128)[0]
    _product_ok(y, _grid(xc)[0], wg, b.detach().cpu())
    _product_ok(dx, _grid(dyc)[0], wg.t().contiguous())
    _product_ok(dw, _grid(dyc.t().contiguous())[0], _grid(xc.t().contiguous())[0])
    want, mag = dyc.double().sum(0), dyc.double().abs().sum(0)
    assert bool(((db.double().cpu() - want).abs() <= 32 * U * mag).all())
    # a frozen weight stands for the same values; up to 16 tokens run another kernel then,
    # whose sums have another order
    f = fp8.quantize(w, square=True, transposed=True)
    y2 = fp8.linear(x, f, b)
    _product_ok(y2, _grid(xc)[0], wg, b.detach().cpu())
    assert torch.equal(dx, torch.autograd.grad(y2, x, dy)[0])
    if M > 16:
        assert torch.equal(y, y2)
    with torch.no_grad():
        assert torch.equal(y2, fp8.linear(x, fp8.quantize(w, square=True), b))
        assert torch.equal(y2, fp8.linear(x, w, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [2, 15, 16])
def test_few_tokens(M, dtype):
    """The kernel that quantises its tokens itself: ragged features, special values."""
    fp8 = _mod()
    x, w = _data(M, 333, dtype, 5), _data(45, 333, torch.float32, 6)
    x[0, 130:260] = 0.0
    wq = fp8.quantize(w.cuda(), square=True)
    b = _data(1, 45, torch.float32, 7)[0]
    _product_ok(fp8.linear(x.cuda(), wq, b.cuda()), _grid(x)[0], _grid(w, 128)[0], b)
    x[1, 332] = math.nan
    y = fp8.linear(x.cuda(), wq).cpu()
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all())


@pytest.mark.gpu
def test_scales_of_any_size_and_special_values():
    fp8 = _mod()
    x, w = torch.randn(40, 300), torch.randn(50, 300)
    x[3] *= 2.0 ** 90
    x[4] *= 2.0 ** -100
    x[5] = 0.0
    x[6, 10], x[7, 20] = math.nan, math.inf
    w[2] = 0.0
    y = fp8.linear(x.cuda(), w.cuda()).cpu()
    keep = [i for i in range(40) if i not in (6, 7)]
    _product_ok(y[keep], _grid(x[keep])[0], _grid(w, 128)[0])
    assert bool(torch.isnan(y[6:8]).all())
    # blocks whose scales' product leaves fp32: zero, not NaN, where the values are zero
    big = torch.zeros(2, 256)
    big[0, 0], big[1, 200] = 2.0 ** 127, 2.0 ** 127
    y = fp8.linear(big.cuda(), torch.stack([big[1], big[0]]).cuda()).cpu()
    assert y[0, 0] == 0 and y[1, 1] == 0
    tiny = torch.full((1, 128), 2.0 ** -120)
    assert fp8.linear(tiny.cuda(), tiny.cuda()).abs().max() == 0


@pytest.mark.gpu
def test_shapes_strides_partial_gradients_and_refusals():
    fp8 = _mod()
    x = torch.randn(3, 5, 64, device="cuda")
    m = fp8.Linear(64, 24).cuda()
    y = m(x)
    assert y.shape == (3, 5, 24)
    assert torch.equal(y.reshape(15, 24), m(x.reshape(15, 64)))
    # views: rows strided, an odd start
    wide = torch.randn(6, 131, device="cuda")
    v = wide[:, 1:65]
    assert torch.equal(m(v), m(v.contiguous()))
    flat = torch.randn(6 * 64 + 1, device="cuda")
    v = flat[1:].view(6, 64)
    assert torch.equal(m(v), m(v.clone()))
    # each subset of gradients
    full = [x.clone().requires_grad_(), m.weight, m.bias]
    dy = torch.randn(3, 5, 24, device="cuda")
    want = torch.autograd.grad(fp8.linear(*full), full, dy)
    for mask in range(1, 8):
        args = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(full)]
        on = [t for t in args if t.requires_grad]
        got = torch.autograd.grad(fp8.linear(*args), on, dy)
        for g, wnt in zip(got, [w for i, w in enumerate(want) if mask >> i & 1]):
            assert torch.equal(g, wnt)
    # the bias alone over a frozen weight, one token without a batch axis, another stream
    bias = m.bias.detach().clone().requires_grad_()
    frozen = fp8.quantize(m.weight, square=True)
    y = fp8.linear(x, frozen, bias)
    assert torch.equal(torch.autograd.grad(y, bias, dy)[0], want[2])
    one = fp8.linear(x[0, 0], frozen, bias)
    assert one.shape == (24,) and torch.equal(one, fp8.linear(x[0, :1], frozen, bias)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = fp8.linear(x, frozen, bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, y)
    # no tokens
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    m.zero_grad()
    m(e).sum().backward()
    assert e.grad.shape == (0, 64) and not m.weight.grad.any() and not m.bias.grad.any()
    with pytest.raises(_lib.AccError):
        fp8.linear(x[..., :60], m.weight)
    with pytest.raises(_lib.AccError):
        fp8.linear(x, m.weight.bfloat16())
    with pytest.raises(_lib.AccError):
        fp8.linear(x.half(), m.weight)
    with pytest.raises(_lib.AccError):
        fp8.linear(x, m.weight, torch.zeros(23, device="cuda"))
    with pytest.raises(_lib.AccError):
        fp8.linear(x, fp8.quantize(m.weight))
    with pytest.raises(_lib.AccError):
        fp8.linear(x.clone().requires_grad_(), fp8.quantize(m.weight, square=True))
    with pytest.raises(_lib.AccError):
        fp8.quantize(torch.empty(0, 8, device="cuda"))
    with pytest.raises(ValueError):
        fp8.quantize(m.weight, transposed=True)


@pytest.mark.gpu
def test_capture_and_repeatability():
    fp8 = _mod()
    x = _data(700, 160, torch.float32, 1).cuda().requires_grad_()
    w = _data(96, 160, torch.float32, 2).cuda().requires_grad_()
    b = torch.zeros(96, device="cuda", requires_grad=True)
    dy = _data(700, 96, torch.float32, 3).cuda()

    def step():
        y = fp8.linear(x, w, b)
        return [y, *torch.autograd.grad(y, [x, w, b], dy)]

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
        for p, q, r in zip(eager, out, again):
            assert torch.equal(p, q) and torch.equal(p, r)
    with torch.no_grad():  # the captured step quantises what the weight holds at replay
        w.mul_(1.37)
    graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(step(), out):
        assert torch.equal(p, q)
