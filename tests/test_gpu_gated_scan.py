"""The gated linear recurrence and its step on the GPU against float64 loops: sizes
around the kernels' tiles, types, layouts, packed sequences, masked and non-finite
values, streams, graphs, and gradients against differences."""

from __future__ import annotations

import pytest
import torch

import ltc_cuda
from _gpu_common import DEV, _native  # noqa: F401
import _seq_ref as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FORMS = ("blend", "decay")


def _gate(shape, form, g, dtype):
    z = torch.randn(shape, generator=g) * 2.0 + 1.0
    if form == "decay":
        z = -torch.nn.functional.softplus(-z)
    return z.clamp(-12, 12).to(dtype)


def _make(N, S, H, form, dtype, gdtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g).to(dtype)
    gate = _gate((N, H), form, g, gdtype)
    state = torch.randn(S, H, generator=g)
    go, gh = torch.randn(N, H, generator=g).to(dtype), torch.randn(S, H, generator=g)
    return x, gate, state, go, gh


def _check(x, gate, state, go, gh, form, runs, call, with_state=True):
    """call(x, gate, state) -> (out, hf) on leaves shaped like the flat tokens."""
    val, tol = R.scan(x, gate, state if with_state else torch.zeros_like(state), form, runs, go, gh)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gate, state)]
    out, hf = call(*leaves[:2], leaves[2] if with_state else None)
    wanted = leaves if with_state else leaves[:2]
    grads = torch.autograd.grad([out, hf], wanted, [go.to(DEV).view(out.shape), gh.to(DEV)])
    for name, got in zip(("out", "hf", "gx", "gg", "gs"), (out.detach(), hf.detach(), *grads)):
        R.close(got, val[name], tol[name], name)
    with torch.no_grad():
        again = call(*leaves[:2], leaves[2] if with_state else None)
    assert torch.equal(again[0], out) and torch.equal(again[1], hf)


def _batch(B, T, H, form, dtype=F32, gdtype=None, with_state=True, seed=0):
    x, gate, state, go, gh = _make(B * T, B, H, form, dtype, gdtype or dtype, seed)
    runs = [(b * T, (b + 1) * T) for b in range(B)]
    _check(x, gate, state, go, gh, form, runs,
           lambda a, b, s: ltc_cuda.ltc_gated_scan(a.view(B, T, H), b.view(B, T, H), s, form=form),
           with_state)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("T", [1, 2, 7, 127, 128, 129, 256, 257, 700])
def test_lengths(T, form):
    _batch(2, T, 33, form)


@pytest.mark.parametrize("H", [1, 3, 8, 31, 32, 63, 64, 65, 130, 1000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_widths(H, dtype):
    _batch(3, 40, H, "blend", dtype)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,gdtype", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_types(dtype, gdtype, form):
    _batch(2, 300, 72, form, dtype, gdtype, with_state=form == "decay")


@pytest.mark.parametrize("B,T", [(24, 8), (300, 1), (1, 1500), (5, 333)])
def test_batches(B, T):
    _batch(B, T, 64, "blend", with_state=B != 24)


def _pack(lengths, before=0, behind=0):
    cu = torch.tensor([before] + [before + sum(lengths[:i + 1]) for i in range(len(lengths))],
                      dtype=torch.int32)
    runs = [(int(cu[i]), int(cu[i + 1])) for i in range(len(lengths))]
    return cu, runs, int(cu[-1]) + behind


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lengths,before,behind", [
    ([5], 0, 0), ([1, 1, 1], 0, 0), ([0, 3, 0, 0, 4, 0], 0, 2), ([300, 1, 0, 255, 257], 0, 0),
    ([128, 128, 256], 0, 130), ([64, 700, 3], 3, 300), ([0, 0], 0, 4), ([0], 0, 0),
    ([2] * 200, 0, 1), ([0] * 70 + [900] + [0] * 70, 0, 0)])
def test_packed(lengths, before, behind, form):
    cu, runs, N = _pack(lengths, before, behind)
    x, gate, state, go, gh = _make(N, len(lengths), 40, form, F32, F32, seed=N)
    # what lies outside the sequences is never looked at
    outside = torch.ones(N, dtype=torch.bool)
    for lo, hi in runs:
        outside[lo:hi] = False
    xn, gn, gon = x.clone(), gate.clone(), go.clone()
    xn[outside] = float("nan")
    gn[outside] = float("inf")
    gon[outside] = float("nan")
    val, tol = R.scan(x, gate, state, form, runs, go, gh)
    leaves = [t.to(DEV).requires_grad_(True) for t in (xn, gn, state)]
    out, hf = ltc_cuda.ltc_gated_scan(*leaves, cu_seqlens=cu.to(DEV), form=form)
    grads = torch.autograd.grad([out, hf], leaves, [gon.to(DEV), gh.to(DEV)])
    for name, got in zip(("out", "hf", "gx", "gg", "gs"), (out.detach(), hf.detach(), *grads)):
        R.close(got, val[name], tol[name], name)


def test_packed_types_and_odd_rows():
    cu, runs, N = _pack([77, 0, 1, 300, 130], 0, 9)
    for dtype, gdtype, H in ((BF16, F32, 37), (F16, F16, 129), (BF16, BF16, 64)):
        x, gate, state, go, gh = _make(N, 5, H, "decay", dtype, gdtype, seed=H)
        _check(x, gate, state, go, gh, "decay", runs,
               lambda a, b, s: ltc_cuda.ltc_gated_scan(a, b, s, cu_seqlens=cu.to(DEV), form="decay"))


def test_boundaries_out_of_order_or_range_stay_in_bounds():
    """Unspecified results, but no access out of range: the buffers around are left alone."""
    x = torch.randn(64, 16, device=DEV)
    gate = torch.zeros(64, 16, device=DEV)
    for cu in ([0, 40, 20, 64], [-5, 10, 64], [0, 10, 1000], [70, 80, 90], [64, 0], [2 ** 31 - 1, -2 ** 31]):
        c = torch.tensor(cu, dtype=torch.int32, device=DEV)
        out, hf = ltc_cuda.ltc_gated_scan(x, gate, None, cu_seqlens=c)
        assert out.shape == x.shape and hf.shape == (len(cu) - 1, 16)
    torch.cuda.synchronize()


@pytest.mark.parametrize("form", FORMS)
def test_empty_calls(form):
    for B, T, H in ((0, 5, 8), (3, 0, 8), (0, 0, 1)):
        x = torch.zeros(B, T, H, device=DEV, requires_grad=True)
        state = torch.randn(B, H, device=DEV, requires_grad=True)
        out, hf = ltc_cuda.ltc_gated_scan(x, x, state, form=form)
        assert out.shape == (B, T, H) and torch.equal(hf, state)
        gh = torch.randn(B, H, device=DEV)
        gx, gs = torch.autograd.grad(hf, [x, state], gh)
        assert gx.shape == x.shape and torch.equal(gs, gh)
        assert torch.equal(ltc_cuda.ltc_gated_scan(x, x, None, form=form)[1], torch.zeros(B, H, device=DEV))


@pytest.mark.parametrize("layout", ["steps", "channels", "offset", "transposed", "expanded_t",
                                    "expanded_b", "reversed_h"])
def test_layouts(layout):
    B, T, H = 3, 150, 24
    g = torch.Generator().manual_seed(7)
    full = torch.randn(2 * B, 2 * T, 2 * H + 1, generator=g).to(DEV)
    views = {"steps": full[:B, ::2, :H], "channels": full[:B, :T, 1:2 * H + 1:2],
             "offset": full[1:B + 1, 1:T + 1, 1:H + 1],
             "transposed": full[:B, :T, :H].permute(1, 0, 2).contiguous().permute(1, 0, 2),
             "expanded_t": full[:B, :1, :H].expand(B, T, H),
             "expanded_b": full[:1, :T, :H].expand(B, T, H),
             "reversed_h": full[:B, :T, :H].permute(0, 2, 1).contiguous().permute(0, 2, 1)}
    v = views[layout]
    gate = (v * 0.5 + 1).requires_grad_(True) if "expanded" not in layout else v.detach()
    want_x = v.contiguous()
    a = ltc_cuda.ltc_gated_scan(v, v, None)
    b = ltc_cuda.ltc_gated_scan(want_x, want_x, None)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # dL/dout in the same layout
    xl, gl = want_x.clone().requires_grad_(True), gate.detach().clone().requires_grad_(True)
    out, hf = ltc_cuda.ltc_gated_scan(xl, gl)
    ga = torch.autograd.grad(out, [xl, gl], v, retain_graph=True)
    gb = torch.autograd.grad(out, [xl, gl], want_x)
    assert torch.equal(ga[0], gb[0]) and torch.equal(ga[1], gb[1])


def test_shared_and_broadcast_leaves_sum_their_gradients():
    B, T, H = 2, 30, 16
    w = torch.randn(H, device=DEV, requires_grad=True)
    x = torch.randn(B, T, H, device=DEV, requires_grad=True)
    out, _ = ltc_cuda.ltc_gated_scan(x, w.expand(B, T, H))
    gw, gx = torch.autograd.grad(out.sum(), [w, x])
    x1 = x.detach().clone().requires_grad_(True)
    g1 = w.detach().expand(B, T, H).contiguous().requires_grad_(True)
    r = torch.autograd.grad(ltc_cuda.ltc_gated_scan(x1, g1)[0].sum(), [g1, x1])
    torch.testing.assert_close(gw, r[0].sum((0, 1)), rtol=1e-5, atol=1e-5)
    assert torch.equal(gx, r[1])
    # one tensor as input and gate
    y = torch.randn(B, T, H, device=DEV, requires_grad=True)
    gy, = torch.autograd.grad(ltc_cuda.ltc_gated_scan(y, y)[0].sum(), [y])
    ya, yb = (y.detach().clone().requires_grad_(True) for _ in range(2))
    ra, rb = torch.autograd.grad(ltc_cuda.ltc_gated_scan(ya, yb)[0].sum(), [ya, yb])
    assert torch.equal(gy, ra + rb)


@pytest.mark.parametrize("form", FORMS)
def test_only_the_wanted_gradients(form):
    x, gate, state, go, gh = (t.to(DEV) for t in _make(60, 2, 20, form, F32, F32))
    full = [t.clone().requires_grad_(True) for t in (x.view(2, 30, 20), gate.view(2, 30, 20), state)]
    out, hf = ltc_cuda.ltc_gated_scan(*full, form=form)
    want = torch.autograd.grad([out, hf], full, [go.view_as(out), gh])
    for i in range(3):
        part = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate(full)]
        out, hf = ltc_cuda.ltc_gated_scan(*part, form=form)
        got, = torch.autograd.grad([out, hf], [part[i]], [go.view_as(out), gh])
        assert torch.equal(got, want[i])
    # through one output only
    out, hf = ltc_cuda.ltc_gated_scan(*full, form=form)
    a = torch.autograd.grad(hf, full, gh, retain_graph=True)
    b = torch.autograd.grad(out, full, go.view_as(out))
    for p, q, r in zip(a, b, want):
        torch.testing.assert_close(p + q, r, rtol=1e-4, atol=1e-5)


def test_non_finite_values_stay_in_their_sequence():
    B, T, H = 4, 200, 8
    x = torch.randn(B, T, H, device=DEV)
    gate = torch.randn(B, T, H, device=DEV)
    x[1, 50, 3] = float("nan")
    x[2, 199, :] = float("inf")
    x = x.requires_grad_(True)
    out, hf = ltc_cuda.ltc_gated_scan(x, gate)
    o = out.detach()
    assert torch.isnan(o[1, 50:, 3]).all() and torch.isfinite(o[1, :50]).all()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[1, 50:, 3] = True
    bad[2, 199] = True
    assert torch.isfinite(o[~bad]).all()
    # the same with the sequences packed end to end
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * T
    op, hp = ltc_cuda.ltc_gated_scan(x.detach().view(B * T, H), gate.view(B * T, H), cu_seqlens=cu)
    assert torch.equal(torch.isfinite(op.view_as(o)), torch.isfinite(o))
    assert torch.equal(op.view_as(o)[~bad], o[~bad])
    # a NaN gradient stays in its sequence too, and before it
    go = torch.ones_like(o)
    go[3, 100, 5] = float("nan")
    xg = torch.randn(B, T, H, device=DEV, requires_grad=True)
    gx, = torch.autograd.grad(ltc_cuda.ltc_gated_scan(xg, gate)[0], [xg], go)
    assert torch.isnan(gx[3, :101, 5]).all() and torch.isfinite(gx[3, 101:]).all()
    assert torch.isfinite(gx[:3]).all()


def test_extreme_gates():
    """Gates of +-inf and the types' largest values: the state is kept, or replaced."""
    T, H = 300, 4
    x = torch.randn(1, T, H, device=DEV)
    h0 = torch.randn(1, H, device=DEV)
    for big in (float("inf"), 3.0e38):
        out, hf = ltc_cuda.ltc_gated_scan(x, torch.full_like(x, big), h0)
        assert torch.equal(out, h0[:, None].expand_as(out)) and torch.equal(hf, h0)
        out, _ = ltc_cuda.ltc_gated_scan(x, torch.full_like(x, -big), h0)
        assert torch.equal(out, x)
        out, _ = ltc_cuda.ltc_gated_scan(x, torch.full_like(x, -big), h0, form="decay")
        assert torch.equal(out, x)
    xg = x.clone().requires_grad_(True)
    gg = torch.full_like(x, float("inf")).requires_grad_(True)
    out, _ = ltc_cuda.ltc_gated_scan(xg, gg, h0)
    for t in torch.autograd.grad(out.sum(), [xg, gg]):
        assert torch.equal(t, torch.zeros_like(t))


@pytest.mark.parametrize("form", FORMS)
def test_gradients_against_differences(form):
    """Central differences of a float64 restatement confirm the reference's formulas, which
    the other tests hold the kernels to."""
    g = torch.Generator().manual_seed(3)
    N, S, H = 9, 3, 2
    runs = [(0, 4), (4, 4), (4, 9)]
    x, state = torch.randn(N, H, generator=g).double(), torch.randn(S, H, generator=g).double()
    gate = _gate((N, H), form, g, torch.float64)
    go, gh = torch.randn(N, H, generator=g).double(), torch.randn(S, H, generator=g).double()
    val, _ = R.scan(x, gate, state, form, runs, go, gh)

    def loss(*a):
        v, _ = R.scan(*a, form, runs)
        return float((v["out"] * go).sum() + (v["hf"] * gh).sum())

    ins = [x, gate, state]
    for i, name in enumerate(("gx", "gg", "gs")):
        for at in range(ins[i].numel()):
            up, dn = [t.clone() for t in ins], [t.clone() for t in ins]
            up[i].view(-1)[at] += 1e-5
            dn[i].view(-1)[at] -= 1e-5
            num = (loss(*up) - loss(*dn)) / 2e-5
            # the difference's own error: 1e-10 h^2 terms and 2^-52 / 2e-5 rounding
            assert abs(num - float(val[name].reshape(-1)[at])) < 1e-8


def test_leaves_edited_in_place_are_an_error_and_second_derivatives_too():
    x = torch.randn(2, 5, 4, device=DEV, requires_grad=True)
    gate = torch.randn(2, 5, 4, device=DEV)
    out, _ = ltc_cuda.ltc_gated_scan(x, gate)
    gate.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out, _ = ltc_cuda.ltc_gated_scan(x, gate)
    g, = torch.autograd.grad(out.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        g.sum().backward()
    out, _ = ltc_cuda.ltc_gated_scan(x, gate)
    out.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()


def test_two_streams_and_a_captured_step():
    x, gate, state, go, gh = (t.to(DEV) for t in _make(4 * 500, 4, 96, "blend", BF16, F32))
    x, gate, go = (t.view(4, 500, 96) for t in (x, gate, go))
    want = ltc_cuda.ltc_gated_scan(x, gate, state)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ltc_cuda.ltc_gated_scan(x, gate, state))
    torch.cuda.synchronize()
    for a in got:
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    leaves = [t.clone().requires_grad_(True) for t in (x, gate, state)]

    def step():
        o, h = ltc_cuda.ltc_gated_scan(*leaves)
        return [o, h, *torch.autograd.grad([o, h], leaves, [go, gh])]

    eager = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = step()
    with torch.cuda.graph(other):
        b = step()
    for i in range(4):
        if i == 2:
            with torch.no_grad():
                leaves[0].mul_(0.5)
            eager = [t.detach().clone() for t in step()]
        graph.replay()
        torch.randn(1000, device=DEV).sum().item()
        other.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(a, b, eager):
            assert torch.equal(p.detach(), r) and torch.equal(q.detach(), r)


def test_capture_beside_a_living_eager_graph_is_an_error():
    """Autograd would tie the default stream into the capture; the node refuses first."""
    x = torch.randn(2, 40, 16, device=DEV, requires_grad=True)
    gate = torch.randn(2, 40, 16, device=DEV)
    go = torch.ones(2, 40, 16, device=DEV)
    alive = ltc_cuda.ltc_gated_scan(x, gate)[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="drop its outputs first"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(ltc_cuda.ltc_gated_scan(x, gate)[0], [x], go)
    want, = torch.autograd.grad(alive, [x], go)
    alive = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ltc_cuda.ltc_gated_scan(x, gate)[0], [x], go)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("B,H,dtype,gdtype", [(1, 64, F32, F32), (1, 1, F32, F32), (3, 37, BF16, F32),
                                              (256, 2048, BF16, BF16), (5, 2500, F16, F32)])
def test_step(B, H, dtype, gdtype, form):
    x, gate, state, _, _ = _make(B, B, H, form, dtype, gdtype, seed=B + H)
    val, tol = R.scan(x, gate, state, form, [(b, b + 1) for b in range(B)])
    st = state.to(DEV)
    out = ltc_cuda.ltc_gated_scan_step(x.to(DEV), gate.to(DEV), st, form=form)
    R.close(out, val["out"], tol["out"], "out")
    R.close(st, val["hf"], tol["hf"], "state")


def test_steps_follow_the_scan():
    B, T, H = 3, 40, 48
    x, gate, state, _, _ = (t.to(DEV) for t in _make(B * T, B, H, "blend", BF16, BF16))
    x, gate = x.view(B, T, H), gate.view(B, T, H)
    out, hf = ltc_cuda.ltc_gated_scan(x, gate, state)
    st = state.clone()
    outs = [ltc_cuda.ltc_gated_scan_step(x[:, t], gate[:, t], st) for t in range(T)]
    val, tol = R.scan(x.reshape(-1, H).cpu(), gate.reshape(-1, H).cpu(), state.cpu(), "blend",
                      [(b * T, (b + 1) * T) for b in range(B)])
    R.close(torch.stack(outs, 1), val["out"], tol["out"], "steps")
    R.close(st, val["hf"], tol["hf"], "state")
    R.close(out, val["out"], tol["out"], "scan")


def test_step_slots():
    P, H = 7, 100
    g = torch.Generator().manual_seed(1)
    state = torch.randn(P, H, generator=g)
    # padding, a slot named three times, one that is not there
    slots = torch.tensor([2, -1, 5, 2, 0, 7, -9, 2, 2 ** 31 - 1], dtype=torch.int32)
    B = slots.numel()
    x, gate = torch.randn(B, H, generator=g), torch.randn(B, H, generator=g)
    st = state.to(DEV)
    out = ltc_cuda.ltc_gated_scan_step(x.to(DEV), gate.to(DEV), st, slots=slots.to(DEV))
    want, wo, tol = state.double().clone(), torch.zeros(B, H).double(), torch.zeros(B, H).double()
    for b, s in enumerate(slots.tolist()):
        if 0 <= s < P:
            v, t = R.scan(x[b:b + 1], gate[b:b + 1], want[s:s + 1], "blend", [(0, 1)])
            want[s] = v["hf"][0]
            wo[b], tol[b] = v["out"][0], 3 * t["out"][0]
        elif s >= P:
            wo[b] = float("nan")
    R.close(out, wo, tol, "out")
    R.close(st, want, 4 * R.UNIT * (1 + want.abs() + 4), "state")
    untouched = [i for i in range(P) if i not in slots.tolist()]
    assert torch.equal(st.cpu()[untouched], state[untouched])
    # states as rows of a wider table
    wide = torch.randn(P, H + 29, generator=g).to(DEV)
    keep = wide.clone()
    o2 = ltc_cuda.ltc_gated_scan_step(x[:3].to(DEV), gate[:3].to(DEV), wide[:, 5:5 + H],
                                      slots=torch.tensor([6, 1, 3], dtype=torch.int32, device=DEV))
    assert torch.equal(wide[:, :5], keep[:, :5]) and torch.equal(wide[:, 5 + H:], keep[:, 5 + H:])
    assert torch.equal(wide[[0, 2, 4, 5]], keep[[0, 2, 4, 5]]) and torch.equal(wide[[6, 1, 3], 5:5 + H], o2)


def test_refusals():
    f = ltc_cuda.ltc_gated_scan
    x = torch.zeros(2, 3, 4, device=DEV)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    for err, call in [
            (ValueError, lambda: f(x, x, form="other")),
            (ValueError, lambda: f(x, x[:, :2])),
            (ValueError, lambda: f(x[0], x[0])),
            (ValueError, lambda: f(x, x, cu_seqlens=cu)),
            (ValueError, lambda: f(x, x, torch.zeros(3, 4, device=DEV))),
            (ValueError, lambda: f(x, x.cpu())),
            (ValueError, lambda: f(x.cpu(), x.cpu())),
            (ValueError, lambda: f(x[..., :0], x[..., :0])),
            (ValueError, lambda: f(x[0], x[0], cu_seqlens=cu.cpu())),
            (ValueError, lambda: f(x[0], x[0], cu_seqlens=cu[:0])),
            (TypeError, lambda: f(x.double(), x.double())),
            (TypeError, lambda: f(x, x.bfloat16())),
            (TypeError, lambda: f(x.bfloat16(), x.half())),
            (TypeError, lambda: f(x, x, torch.zeros(2, 4, device=DEV, dtype=torch.float16))),
            (TypeError, lambda: f(x[0], x[0], cu_seqlens=cu.long()))]:
        with pytest.raises(err):
            call()
    s = ltc_cuda.ltc_gated_scan_step
    y, st = x[:, 0], torch.zeros(2, 4, device=DEV)
    sl = torch.zeros(2, dtype=torch.int32, device=DEV)
    for err, call in [
            (ValueError, lambda: s(x, x, st)),
            (ValueError, lambda: s(y, y, torch.zeros(3, 4, device=DEV))),
            (ValueError, lambda: s(y, y, torch.zeros(4, 2, device=DEV).t())),
            (ValueError, lambda: s(y, y, torch.zeros(1, 4, device=DEV).expand(2, 4))),
            (ValueError, lambda: s(y, y, st, slots=sl[:1])),
            (ValueError, lambda: s(y, y, st, form="x")),
            (TypeError, lambda: s(y, y, st, slots=sl.long())),
            (TypeError, lambda: s(y, y, st.half())),
            (RuntimeError, lambda: s(y.clone().requires_grad_(True), y, st))]:
        with pytest.raises(err):
            call()
