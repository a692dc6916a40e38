"""gloo gets CPU tensors only. Its collectives on device tensors have hung where several ranks
share a GPU; accunet.dist copies device tensors to host memory first, synchronously."""
import os

import pytest
import torch
from test_dist_gpu import HERE, _run


class _Device:
    """What accunet.dist asks of a device tensor, over a CPU tensor."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def cpu(self):
        return self.t.clone()

    def copy_(self, h):
        self.t.copy_(h)


def test_collectives_of_device_tensors_go_through_the_host(monkeypatch):
    from accunet import dist as adist
    seen = []
    monkeypatch.setattr(adist.dist, "all_reduce", lambda t, **kw: (seen.append(t), t.mul_(3))[0])
    monkeypatch.setattr(adist.dist, "broadcast", lambda t, src, **kw: (seen.append(t), t.add_(1))[0])
    monkeypatch.setattr(adist.dist, "get_backend", lambda group=None: "gloo")
    d = _Device(torch.ones(4))
    assert adist.all_reduce(d, async_op=True) is None and torch.equal(d.t, torch.full((4,), 3.0))
    adist.broadcast(d, 0)
    assert torch.equal(d.t, torch.full((4,), 4.0))
    assert all(isinstance(t, torch.Tensor) for t in seen) and len(seen) == 2
    # CPU tensors, and device tensors over RCCL, as they are
    t = torch.ones(2)
    adist.all_reduce(t)
    assert seen[-1] is t
    monkeypatch.setattr(adist.dist, "get_backend", lambda group=None: "nccl")
    monkeypatch.setattr(adist.dist, "all_reduce", lambda t, **kw: seen.append(t) or "work")
    assert adist.all_reduce(d, async_op=True) == "work" and seen[-1] is d


@pytest.mark.gpu
@pytest.mark.parametrize("world", [2, 4, 8])
def test_no_device_tensor_reaches_gloo(world):
    """The data-parallel runs and checks of dist_worker.py (2, 4 and 8 ranks on the one GPU;
    three of its modes with 8)."""
    modes = {} if world < 8 else {"DIST_MODES": "graph,eager,graph_wire16"}  # a minute otherwise
    r = _run([os.path.join(HERE, "gloo_host_worker.py")], nproc=world, timeout=110,
             threads=2 if world == 8 else 4, **modes)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    assert "DIST_OK" in r.stdout and r.stdout.count("HOST_OK") == world
    print("\n".join(l for l in r.stdout.splitlines() if "fp64 mean" in l or "HOST_OK" in l))
