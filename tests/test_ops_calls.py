"""How the public operators are called: under a tracer, with forward-mode derivatives, while a graph is captured, from several threads."""
import os
import subprocess
import sys
import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from lsdm_amd import _lib, ops

gpu = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


def calls(device):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(device)
    x, w, b, res, n = r(70, 16), r(8, 16), r(8), r(70, 8), r(16)
    return x, [lambda t: ops.linear(t, w), lambda t: ops.linear(x, w, b, "gelu", residual=t @ w.t()), lambda t: ops.linear(res, t[:, :8].contiguous()),
               lambda t: ops.layer_norm(t), lambda t: ops.layer_norm(x, t[0].contiguous(), n)]


def refuse_tracing(device):
    x, forms = calls(device)
    packed = lambda t: ops.checkpoint8(t).codes
    for f in [*forms, packed]:
        with pytest.raises(_lib.LsdmError, match="traced"):
            torch.jit.trace(f, (x,))
        with pytest.raises(_lib.LsdmError, match="traced"):
            make_fx(f)(x)


def refuse_forward_mode(device):
    x, forms = calls(device)
    for f in forms:
        with forward_ad.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(_lib.LsdmError, match="forward-mode"):
                    f(forward_ad.make_dual(x, torch.ones_like(x)))


def test_traced_calls_are_refused_on_the_host():
    refuse_tracing("cpu")


@gpu
def test_traced_calls_are_refused():
    """A tracer records tensors' operations, and these kernels write through pointers: the recorded graph would return memory that nothing wrote."""
    refuse_tracing(DEV)
    c = ops.checkpoint8(torch.randn(3, 40, device=DEV))
    with pytest.raises(_lib.LsdmError, match="traced"):
        torch.jit.trace(lambda t: ops.Checkpoint8(t, c.exps, c.shape, c.dtype).restore(), (c.codes,))
    x, forms = calls(DEV)
    for f in forms:
        assert torch.equal(f(x), f(x))                      # and are what they were afterwards
    t = x.clone().requires_grad_(True)
    for f in (forms[0], forms[3]):
        y = f(t)
        dy = torch.randn_like(y)
        want = torch.autograd.grad(y, [t], dy, retain_graph=True)[0]
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda g: torch.autograd.grad(y, [t], g, retain_graph=True)[0])(dy)
        assert torch.equal(torch.autograd.grad(y, [t], dy)[0], want)


def test_forward_mode_is_refused_on_the_host():
    refuse_forward_mode("cpu")


@gpu
def test_forward_mode_is_refused():
    refuse_forward_mode(DEV)
    x, forms = calls(DEV)
    with forward_ad.dual_level():
        for f in forms:                                     # a dual number elsewhere does not matter
            d = forward_ad.make_dual(torch.ones(3, device=DEV), torch.ones(3, device=DEV))
            assert torch.equal(f(x), f(x)) and forward_ad.unpack_dual(d).tangent is not None


@gpu
def test_capture_with_a_live_eager_graph_behind_the_inputs_is_refused():
    """The captured call's inputs are not the leaves themselves but computed from them inside the capture (a cast, a slice, a tied weight): the backward
    pass would end at the leaves' gradient nodes on the default stream all the same."""
    w = torch.randn(8, 16, device=DEV, requires_grad=True)
    n = torch.ones(16, device=DEV, requires_grad=True)
    b = torch.zeros(8, device=DEV, requires_grad=True)
    x = torch.randn(70, 16, device=DEV)
    alive = [ops.linear(x, w, b), ops.layer_norm(x, n)]     # built on the default stream
    own = torch.randn(8, 16, device=DEV, requires_grad=True)    # a leaf no eager graph holds
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    refused, taken = [], []
    with torch.cuda.graph(g, stream=s):
        for f in (lambda: ops.linear(x.half(), w.half()), lambda: ops.linear(x, w[:4]), lambda: ops.linear(x, w.detach(), b * 2), lambda: ops.layer_norm(x, n * 0.5),
                  lambda: ops.layer_norm(ops.linear(x[:, :8].contiguous(), (w.t() + 1.0).contiguous())), lambda: ops.layer_norm((x + n).view(7, 10, 16))):
            try:
                f()
            except _lib.LsdmError as e:
                refused.append(str(e))
        y = ops.linear(x.half(), own.half() * 2, w.detach()[:, 0])
        taken += [y, *torch.autograd.grad(y, [own], torch.ones_like(y))]
    assert len(refused) == 6 and all("live autograd graph" in r for r in refused)
    y = ops.linear(x.half(), own.half() * 2, w.detach()[:, 0])
    want = [y, *torch.autograd.grad(y, [own], torch.ones_like(y))]
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(taken, want))
    torch.autograd.grad(alive[0], [w, b], torch.ones_like(alive[0]))      # the eager graphs are as they were
    torch.autograd.grad(alive[1], [n], torch.ones_like(alive[1]))


def test_first_calls_of_several_threads_load_one_front_end():
    """In a process of its own, with threads that change places at every step."""
    code = """
import sys, threading
sys.setswitchinterval(1e-6)
import torch
from lsdm_amd import _lib
at, found = threading.Barrier(8), []
def run():
    at.wait()
    found.append(id(_lib.load_torch_ops()))
threads = [threading.Thread(target=run) for _ in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(found) == 8 and len(set(found)) == 1, found
"""
    for _ in range(3):
        subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=120)


@gpu
def test_calls_from_several_threads():
    """Every thread on a stream of its own, forward and backward, with refused calls in between: the results of one thread alone."""
    gen = torch.Generator().manual_seed(1)
    sets = []
    for k in range(4):
        r = lambda *s: torch.randn(*s, generator=gen).to(DEV).bfloat16()
        sets.append([r(300 + 41 * k, 72), r(88, 72), r(88), r(300 + 41 * k, 88), r(88), r(300 + 41 * k, 88)])

    def work(v):
        x, w, b, res, n, dy = (t.clone().requires_grad_(True) for t in v)
        y = ops.layer_norm(ops.linear(x, w, b, "silu", res), n)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b, res, n], dy.detach())]
    want = [work(v) for v in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(k):
        s = torch.cuda.Stream()
        with torch.enable_grad(), torch.cuda.stream(s):
            for i in range(6):
                got = work(sets[k])
                with pytest.raises(ValueError, match="eps"):
                    ops.layer_norm(sets[k][0], eps=-1.0 - k)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    wrong.append((k, i))
    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
