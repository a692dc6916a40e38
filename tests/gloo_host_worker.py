"""One rank of tests/test_gloo_host.py: the run of dist_worker.py with every collective watched.
gloo gets CPU tensors only; a device tensor that would reach it raises before the call. The
worker's own all_gather of its results goes through host memory here."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def watched(fn):
    def call(tensor, *args, **kw):
        if tensor.is_cuda and dist.get_backend(kw.get("group")) == "gloo":
            raise RuntimeError(f"gloo {fn.__name__} of a device tensor")
        calls[fn.__name__] = calls.get(fn.__name__, 0) + 1
        return fn(tensor, *args, **kw)
    return call


def gathered(fn):
    def call(outs, tensor, *args, **kw):
        host = [torch.empty(t.shape, dtype=t.dtype) for t in outs]
        fn(host, tensor.cpu(), *args, **kw)
        for t, h in zip(outs, host):
            t.copy_(h)
    return call


calls = {}
dist.all_reduce, dist.broadcast = watched(dist.all_reduce), watched(dist.broadcast)
dist.all_gather = gathered(dist.all_gather)

import dist_worker  # noqa: E402

dist_worker.main()
assert calls["all_reduce"] > 0 and calls["broadcast"] > 0, calls
print(f"HOST_OK {calls}", flush=True)
