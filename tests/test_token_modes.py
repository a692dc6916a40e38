"""The token-block operators under torch's forward mode and under a trace, without a backward:
forward mode is refused (there is no such derivative), a trace records the operator and not
the empty outputs that its kernel fills. On the CPU, with torch operations in the place of the
launches; the same calls on the GPU."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from accunet import blocknorm, distill, fp8, kern

gpu = pytest.mark.gpu


def _launches_on_the_host(monkeypatch):
    """Stand-ins that write through the tensors' memory, as a launch does."""
    def norm(x, f, w1, b1, s, g, w2, b2, layer, eps, r, h, stats, P, L, C):
        v = x.numpy() if f is None else x.numpy() + f.numpy()
        if r is not None:
            r.numpy()[...] = v
        if h is not None:
            d = v - v.mean(-1, keepdims=True)
            h.numpy()[...] = d / np.sqrt((d * d).mean(-1, keepdims=True) + eps)

    def linear(x, w, wq, wqs, bias, y, need_w, need_wt, M, N, K):
        v = w.numpy() if w is not None else np.ones((N, K), np.float32)
        y.numpy()[...] = x.numpy() @ v.T + bias.numpy()

    def loss(z, idx, top, rest, out, *a):
        out.numpy()[...] = np.square(z.numpy()).sum()

    def quantize(x, square, q, s, qt, st, R, C):
        s.numpy()[...] = 127

    monkeypatch.setattr(kern, "_check", lambda *a, **k: None)
    monkeypatch.setattr(kern, "blocknorm_fwd", norm)
    monkeypatch.setattr(kern, "fp8_linear_fwd", linear)
    monkeypatch.setattr(kern, "fp8_quantize", quantize)
    monkeypatch.setattr(kern, "distill_fwd", loss)


def _calls(dev):
    g = torch.Generator().manual_seed(0)
    w, b = torch.randn(24, 16, generator=g).to(dev), torch.randn(24, generator=g).to(dev)
    f = torch.randn(6, 16, generator=g).to(dev)
    idx = torch.randint(0, 16, (6, 3), generator=g).to(dev)
    top = torch.randn(6, 3, generator=g).to(dev)
    with torch.no_grad():
        wq = fp8.quantize(w, square=True)
    return {"norm": lambda x: blocknorm.norm(x, kind="layer"),
            "sandwich": lambda x: blocknorm.sandwich_norm(x, f)[1],
            "linear": lambda x: fp8.linear(x, w, b),
            "frozen": lambda x: fp8.linear(x, wq, b),
            "distill": lambda x: distill.topk_distill(x, idx, top)}


def _inputs(dev):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(6, 16, generator=g).to(dev) for _ in range(3)]


def _refuses_forward_mode(name, dev):
    call = _calls(dev)[name]
    x, t, _ = _inputs(dev)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            with pytest.raises(RuntimeError):
                call(fwAD.make_dual(x, t))


def _is_traced(name, dev):
    call = _calls(dev)[name]
    x, y, z = _inputs(dev)
    with torch.no_grad():
        traced = torch.jit.trace(call, x, check_trace=False)
        for v in (x, y, z):
            junk = torch.full((1 << 12,), float("nan"), device=dev)  # what freed memory holds
            del junk
            assert torch.equal(traced(v), call(v))
        # more rows than were traced: their own sizes, or refused beside a tensor of fewer
        more = torch.cat([x, y[:3]])
        if name in ("sandwich", "distill"):
            with pytest.raises(Exception, match="differ|must have"):
                traced(more)
        else:
            assert torch.equal(traced(more), call(more))


NAMES = ["norm", "sandwich", "linear", "frozen", "distill"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_on_the_host(name, monkeypatch):
    _launches_on_the_host(monkeypatch)
    _refuses_forward_mode(name, "cpu")


@pytest.mark.parametrize("name", NAMES)
def test_trace_on_the_host(name, monkeypatch):
    _launches_on_the_host(monkeypatch)
    _is_traced(name, "cpu")


@gpu
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode(name):
    _refuses_forward_mode(name, "cuda")


@gpu
@pytest.mark.parametrize("name", NAMES)
def test_trace(name):
    _is_traced(name, "cuda")
