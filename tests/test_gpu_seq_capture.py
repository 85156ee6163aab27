"""Captured backward passes of the modules on the sequence and token operators, beside
autograd graphs of the same parameters that are still alive."""

from __future__ import annotations

import pytest
import torch

import ltc
import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _layer():
    torch.manual_seed(4)
    m = ltc.LinearTimeConstant(6, 16).to(DEV)
    x = torch.randn(2, 150, 6, device=DEV)
    return list(m.parameters()), lambda v: m(v)[0], x


def _scan():
    x, gate = (torch.randn(2, 150, 8, device=DEV, requires_grad=True) for _ in range(2))
    return [x, gate], lambda v: ltc_cuda.ltc_gated_scan(v, gate)[0], x


def _readout(which):
    torch.manual_seed(5)
    m = ltc.TokenReadout(16, 300).to(DEV)
    h = torch.randn(4, 16, device=DEV)
    ids = torch.randint(0, 300, (4,), device=DEV)
    if which == "log_probs":
        return [m.proj.weight], lambda v: m.log_probs(v, ids)[0], h
    t = torch.randn(4, 3, device=DEV)
    tid = torch.randint(0, 300, (4, 3), device=DEV)
    return [m.proj.weight], lambda v: m.distill(v, t, tid), h


MAKE = {"scan": _scan, "layer": _layer, "log_probs": lambda: _readout("log_probs"),
        "distill": lambda: _readout("distill")}


def _captured(leaves, f, x):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(x)
        grads = torch.autograd.grad(out, leaves, torch.ones_like(out), allow_unused=True)
    return graph, grads


def _replays_are(graph, got, want):
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert len(got) == len(want)
        for a, b in zip(got, want):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
        torch.randn(1000, device=DEV).sum().item()


@pytest.mark.parametrize("what", MAKE)
def test_an_eager_graph_of_the_parameters_is_an_error(what):
    """A module's parameters lie behind other nodes of the graph, not on the operator's edges."""
    leaves, f, x = MAKE[what]()
    alive = f(x)
    with pytest.raises(RuntimeError, match="drop its outputs first"):
        _captured(leaves, f, x)
    torch.cuda.synchronize()
    want = torch.autograd.grad(alive, leaves, torch.ones_like(alive), allow_unused=True)
    alive = None
    graph, got = _captured(leaves, f, x)
    _replays_are(graph, got, want)


def test_parameters_that_the_pass_does_not_reach_may_have_one():
    leaves, f, x = _layer()
    alive = f(x)
    y = x.clone().requires_grad_(True)
    want = torch.autograd.grad(f(y), [y], torch.ones_like(alive))
    graph, got = _captured([y], f, y)
    _replays_are(graph, got, want)
    del alive


@pytest.mark.parametrize("what", MAKE)
def test_a_warm_up_on_another_stream_may_live_on(what):
    """torch's recipe for whole-network capture keeps its last loss."""
    leaves, f, x = MAKE[what]()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            out = f(x)
            want = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True,
                                       allow_unused=True)
    torch.cuda.current_stream().wait_stream(side)
    graph, got = _captured(leaves, f, x)
    _replays_are(graph, got, want)
    del out
