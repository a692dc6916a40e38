"""Kernel forms of the token-block operators that only large calls take, against 64 bits: the
8-bit product in 256 x 256 tiles over many scale groups, and distillation rows of more vectors
than are marked at once, with gradients stored past the caches. Tolerances: those of
test_fp8.py and test_distill.py."""
import pytest
import torch
from test_distill import U, _close, _fn, _reference
from test_fp8 import _data, _product_ok


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(4096, 4100, 1300), (1300, 4100, 4096), (4099, 1300, 4096)])
def test_products_in_large_tiles(M, N, K, dtype):
    """272 tiles of 256 x 256 and 11 k-tiles: y, dw and dx of the three sizes, in this order.
    The quantised values themselves are checked bit for bit in test_fp8.py."""
    from accunet import fp8
    x, w = _data(M, K, dtype, 1).cuda(), _data(N, K, torch.float32, 2).cuda()
    b, dy = _data(1, N, torch.float32, 3)[0].cuda(), _data(M, N, dtype, 4).cuda()
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = fp8.linear(x, w, b)
    dx, dw, _ = torch.autograd.grad(y, leaves, dy)
    xd, wd = x.detach(), w.detach()

    def val(t, square=False):
        return fp8.quantize(t.contiguous(), square=square).values().double()

    wv = val(wd, True)
    _product_ok(y, val(xd), wv, b.detach())
    _product_ok(dx, val(dy), wv.t().contiguous())
    _product_ok(dw, val(dy.t()), val(xd.t()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V", [(torch.bfloat16, 300, 128000), (torch.bfloat16, 258, 131101),
                                       (torch.float32, 260, 65413), (torch.float32, 256, 66001)])
@pytest.mark.parametrize("has_rest", [False, True])
def test_long_distillation_rows(R, V, dtype, has_rest):
    """64 MB of logits and more; up to 16384 vectors a row, and beyond."""
    K = 64
    g = torch.Generator().manual_seed(6)
    z = (3 * torch.randn(R, V, generator=g)).to(dtype)
    idx = (torch.randint(0, V, (R, 1), generator=g) + (V // K) * torch.arange(K)) % V
    idx[:, 1] = (idx[:, 0] + 1) % V  # neighbours of one vector, or of two
    top = (2 * torch.randn(R, K, generator=g)).to(dtype)
    idx[2, 5:] = -1
    idx[3] = -1
    r = torch.rand(R, generator=g) * 0.6 if has_rest else None
    pick = [0, 1, 2, 3, R // 2, R - 1]
    want, dwant, tl, td, _ = _reference(z[pick], idx[pick], top[pick], r[pick] if has_rest else None, 1.7)
    zd = z.cuda().requires_grad_()
    kw = dict(rest=r.cuda() if has_rest else None, temperature=1.7)
    per = _fn()(zd, idx.cuda(), top.cuda(), reduction="none", **kw)
    _close(per[pick], want, tl, "loss")
    for loss, n in ((per, 1), (_fn()(zd, idx.cuda(), top.cuda(), **kw), R - 1)):
        (dz,) = torch.autograd.grad(loss, zd, torch.ones_like(loss))
        _close(dz[pick], dwant / n, (td + 8 * U * dwant.abs()) / n, "dz")
        del dz
