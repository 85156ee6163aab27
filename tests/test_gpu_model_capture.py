"""The token model's operators in captured graphs: replays against eager results, two
graphs side by side, and captures beside autograd graphs that are still alive."""

from __future__ import annotations

import pytest
import torch

import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rand(*shape):
    return torch.randn(*shape, device=DEV)


def _conv(T=70):
    x, w, b = _rand(2, T, 24).requires_grad_(True), _rand(24, 4).requires_grad_(True), _rand(24).requires_grad_(True)
    return [x, w, b], lambda: ltc_cuda.ltc_causal_conv(x, w, b, activation="silu")[0], x


def _ssm(T=200):
    """Cut into chunks, so that states pass through the workspace."""
    x, d = _rand(1, T, 8).requires_grad_(True), (torch.rand(1, T, 8, device=DEV)).requires_grad_(True)
    A = (-torch.rand(8, 16, device=DEV)).requires_grad_(True)
    B, C = _rand(1, T, 16).requires_grad_(True), _rand(1, T, 16).requires_grad_(True)
    return [x, d, A, B, C], lambda: ltc_cuda.ltc_selective_scan(x, d, A, B, C)[0], x


def _embed(n=9000):
    t = _rand(500, 16).requires_grad_(True)
    ids = torch.randint(0, 500, (n,), device=DEV)
    return [t], lambda: ltc_cuda.ltc_embed(t, ids, 2.0), t


MAKE = {"conv": _conv, "ssm": _ssm, "embed": _embed}


def _step(leaves, f):
    out = f()
    return [out, *torch.autograd.grad(out, leaves, torch.ones_like(out))]


def _capture(leaves, f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(leaves, f)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = _step(leaves, f)
    return graph, [r.detach() for r in res]


@pytest.mark.parametrize("kind", list(MAKE))
def test_replays(kind):
    leaves, f, x = MAKE[kind]()
    graph, got = _capture(leaves, f)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        kept = [g.clone() for g in got]
        want = [w.detach() for w in _step(leaves, f)]
        assert all(torch.equal(a, b) for a, b in zip(kept, want)), k


@pytest.mark.parametrize("kind", list(MAKE))
def test_two_graphs(kind):
    """Each has its own workspace: replayed at once on two streams they are right."""
    pairs = [MAKE[kind]() for _ in range(2)]
    graphs = [_capture(leaves, f) for leaves, f, _ in pairs]
    want = [[w.detach().clone() for w in _step(leaves, f)] for leaves, f, _ in pairs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, got), ref in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("kind", list(MAKE))
def test_capture_beside_an_eager_graph_is_refused(kind):
    leaves, f, _ = MAKE[kind]()
    alive = f()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            _step(leaves, f)
    torch.cuda.synchronize()
    del alive
    graph, got = _capture(leaves, f)
    graph.replay()
    torch.cuda.synchronize()
    kept = [g.clone() for g in got]
    assert all(torch.equal(a, b.detach()) for a, b in zip(kept, _step(leaves, f)))


def test_decode_step_in_a_graph():
    """Convolution, scan and adjustments of one token, states updated in place by replays."""
    B, H, N, V = 5, 24, 8, 300
    w, A = _rand(H, 4), -torch.rand(H, N, device=DEV)
    table = _rand(V, H)
    ids, seen = torch.zeros(B, dtype=torch.int64, device=DEV), torch.randint(0, V, (B, 12), device=DEV)
    tail, state = torch.zeros(B, 3, H, device=DEV), torch.zeros(B, H, N, device=DEV)
    slots = torch.tensor([3, -1, 0, 4, 1], dtype=torch.int32, device=DEV)

    @torch.no_grad()
    def step(tail, state):
        x = ltc_cuda.ltc_embed(table, ids)
        x = ltc_cuda.ltc_causal_conv_step(x, w, tail, slots=slots, activation="silu")
        y = ltc_cuda.ltc_selective_scan_step(x, x, A, x[:, :N], x[:, N:2 * N], state, slots=slots,
                                             delta_softplus=True)
        return ltc_cuda.ltc_adjust_logits(y @ table.t(), seen, repetition=1.2, frequency=0.1)

    step(tail.clone(), state.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(tail, state)
    tail2, state2 = tail.clone(), state.clone()
    for k in range(5):
        ids.copy_(torch.randint(0, V, (B,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        want = step(tail2, state2)
        assert torch.equal(out, want) and torch.equal(tail, tail2) and torch.equal(state, state2)


def test_another_device_is_named_by_the_tensors():
    """Work goes to the tensors' device, whatever the current one is."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    x = torch.randn(2, 30, 8, device="cuda:1")
    w = torch.randn(8, 4, device="cuda:1")
    with torch.cuda.device(0):
        out = ltc_cuda.ltc_causal_conv(x, w)[0]
    assert out.device == x.device
