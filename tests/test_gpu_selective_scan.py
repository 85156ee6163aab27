"""The selective scan against its definition in 64 bits, token by token: lengths from none
to several chunks, states that do not fill a wave's four, groups, packed sequences; its
gradients, and its step.

Tolerances count roundings of 2^-24, relative to the sums of the terms' sizes (the same
formulas over absolute values, _sizes). A step of the recurrence takes the product s A
log2(e) (two roundings, which an exponential turns into |s A| of them: at most 4 here), the
exponential (2), a product and a multiply-add: with the step size's own error of at most 8
steps, carried by the exponent as |s A| too, 40 a token at most, and they add up over the
tokens that a value has come through: 40 L for the longest sequence L. The gates at the end
add 16. Outputs of 16 bits are off by half a step of their own besides."""

from __future__ import annotations

import pytest
import torch

import _model_ref as R
import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
NAMES = ("x", "delta", "A", "B", "C", "D", "z", "bias", "state")


def _inputs(lead, rows, H, N, G, dtype, skip, gated, softplus, state, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    dt = R.TYPES[dtype]
    t = {"x": rand(*lead, H).to(dt), "A": -torch.rand(H, N, generator=g) * 3 - 0.1,
         "B": rand(*lead, G, N).to(dt), "C": rand(*lead, G, N).to(dt),
         "D": rand(H) if skip else None, "z": rand(*lead, H).to(dt) if gated else None,
         "state": rand(rows, H, N) if state else None}
    if softplus:
        t["bias"] = rand(H) - 1.0
        t["delta"] = rand(*lead, H).to(dt)
    else:
        t["bias"] = None
        t["delta"] = (torch.rand(*lead, H, generator=g) * 0.5 + 0.01).to(dt)
    return t


def _sizes(t, cu, softplus, go, gh):
    """Sums of the terms' sizes of out, state_final and every gradient."""
    a = {k: None if v is None else v.double() for k, v in t.items()}
    A = a["A"]
    H, N = A.shape
    G = a["B"].shape[-2]
    res = {k: torch.zeros_like(v) for k, v in a.items() if v is not None}
    out = torch.zeros_like(a["x"])
    n = a["x"].shape[0] if cu is None else cu.numel() - 1
    hf = a["x"].new_zeros(n, H, N)

    def wide(v):
        return v.abs().repeat_interleave(H // G, 0)

    for s, of in R.runs_of(a["x"], cu):
        L = of(a["x"]).shape[0]
        h = A.new_zeros(H, N) if a["state"] is None else a["state"][s].abs()
        hs, size, slope = [h], [], []
        for i in range(L):
            v = of(a["delta"])[i] + (0 if a["bias"] is None else a["bias"])
            d = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v.abs()
            size.append(d)
            slope.append(torch.sigmoid(v) if softplus else torch.ones_like(v))
            h = torch.exp(d[:, None] * A) * h + (d * of(a["x"])[i].abs())[:, None] * wide(of(a["B"])[i])
            hs.append(h)
        hf[s] = h
        g = gh[s].double().abs()
        for i in reversed(range(L)):
            x, B, C, d = of(a["x"])[i].abs(), wide(of(a["B"])[i]), wide(of(a["C"])[i]), size[i]
            y = (hs[i + 1] * C).sum(-1) + (0 if a["D"] is None else a["D"].abs() * x)
            o = of(go)[i].double().abs()
            dy = o
            if a["z"] is not None:
                z = of(a["z"])[i]
                dy = o * R.silu(z).abs()
                of(res["z"])[i] += o * y * 1.1
                of(out)[i] += y * R.silu(z).abs()
            else:
                of(out)[i] += y
            e = g + dy[:, None] * C
            of(res["C"])[i] += (hs[i + 1] * dy[:, None]).view(G, H // G, N).sum(1)
            of(res["B"])[i] += (e * (d * x)[:, None]).view(G, H // G, N).sum(1)
            g = torch.exp(d[:, None] * A) * e
            k = g * hs[i]
            s1 = (e * B).sum(-1)
            of(res["x"])[i] += d * s1
            dd = x * s1 + (k * A.abs()).sum(-1)
            of(res["delta"])[i] += dd * slope[i]
            res["A"] += k * d[:, None]
            if a["D"] is not None:
                of(res["x"])[i] += a["D"].abs() * dy
                res["D"] += dy * x
            if a["bias"] is not None:
                res["bias"] += dd * slope[i]
        if a["state"] is not None:
            res["state"][s] += g
    return out, hf, res


def _close(got, want, mag, dtype, count, what):
    got, want = got.detach().cpu().double(), want.detach()
    err = count * U * mag
    tol = err + (R.half_step(dtype) * (want.abs() + err) if dtype != "fp32" else U * want.abs())
    tol = tol + torch.finfo(R.TYPES[dtype]).tiny
    off = (got - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), (what, float((off / tol).max()))


def _call(t, cu, softplus):
    B, C = t["B"], t["C"]
    if B.shape[-2] == 1:
        B, C = B.squeeze(-2), C.squeeze(-2)
    return ltc_cuda.ltc_selective_scan(t["x"], t["delta"], t["A"], B, C, t["D"], t["z"], t["bias"],
                                       t["state"], None if cu is None else cu.to(DEV), softplus)


def _check(lead, cu, H, N, G, dtype, skip, gated, softplus, state, seed=0):
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    rows = lead[0] if cu is None else len(cu) - 1
    t = _inputs(lead, rows, H, N, G, dtype, skip, gated, softplus, state, seed)
    g = torch.Generator().manual_seed(seed + 50)
    go = torch.randn(*lead, H, generator=g).to(R.TYPES[dtype])
    gh = torch.randn(rows, H, N, generator=g)
    d = {k: None if v is None else v.double().requires_grad_(True) for k, v in t.items()}
    want, hf = R.scan(d["x"], d["delta"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"], d["state"],
                      c, softplus)
    names = [k for k in NAMES if d[k] is not None]
    ref = R.gradients([want, hf], [go.double(), gh.double()], [d[k] for k in names])
    mo, mh, mg = _sizes(t, c, softplus, go, gh)
    dev = {k: None if v is None else v.to(DEV).requires_grad_(True) for k, v in t.items()}
    out, fin = _call(dev, c, softplus)
    long = max([lead[-1] if cu is None else 0] + ([] if cu is None else
                                                 [b - a for a, b in zip(cu, cu[1:])]))
    count = 40 * long + 16 + N
    _close(out, want, mo, dtype, count, "out")
    _close(fin, hf, mh, "fp32", count, "state")
    got = torch.autograd.grad([out, fin], [dev[k] for k in names], [go.to(DEV), gh.to(DEV)])
    tokens = want.numel() // H
    for k, a, r in zip(names, got, ref):
        # sums over channels or tokens add a rounding a term at most
        more = 2 * count + 32 + (H if k in "BC" else 0) + (tokens if k in ("A", "D", "bias") else 0)
        _close(a, r, mg[k], "fp32" if a.dtype == torch.float32 else dtype, more, k)
    with torch.no_grad():
        plain, pf = _call(dev, c, softplus)
    assert torch.equal(plain, out) and torch.equal(pf, fin)


@pytest.mark.parametrize("lead,cu", [
    ((2, 1), None), ((3, 15), None), ((1, 16), None), ((2, 17), None), ((2, 40), None),
    ((1, 150), None), ((3, 0), None), ((0, 4), None), ((50,), [0, 20, 20, 21, 45]),
    ((90,), [3, 3, 35, 80]), ((16,), [0, 16]), ((20,), [20, 20]), ((9,), [0, 0]), ((5,), [2])])
@pytest.mark.parametrize("H,N,G,dtype,skip,gated,softplus,state", [
    (6, 16, 1, "fp32", True, True, True, True), (70, 4, 1, "bf16", True, False, True, False),
    (12, 5, 3, "fp32", False, True, False, True), (8, 1, 2, "fp16", True, True, True, False)])
def test_lengths(lead, cu, H, N, G, dtype, skip, gated, softplus, state):
    _check(lead, cu, H, N, G, dtype, skip, gated, softplus, state)


@pytest.mark.parametrize("N", [1, 2, 3, 4, 7, 8, 13, 16, 24, 31, 32, 33, 40, 63, 64])
@pytest.mark.parametrize("dtype,gated", [("fp32", True), ("bf16", False)])
def test_states(N, dtype, gated):
    _check((2, 35), None, 5, N, 1, dtype, True, gated, True, True)
    _check((40,), [1, 17, 17, 36], 4, N, 2, dtype, False, gated, False, True)


@pytest.mark.parametrize("H,G", [(1, 1), (63, 1), (64, 1), (65, 1), (130, 2), (129, 3), (200, 1)])
def test_channels(H, G):
    _check((1, 33), None, H, 6, G, "fp32", True, True, True, True)
    _check((70,), [0, 30, 66], H, 4, G, "bf16", True, False, True, False)


@pytest.mark.parametrize("T", [63, 64, 65, 128, 200, 330])
def test_chunks(T):
    """Long sequences of few channels are cut; packed ones with boundaries in the chunks."""
    _check((1, T), None, 3, 4, 1, "fp32", True, True, True, True)
    _check((T,), [0, 5, T // 2, T // 2, T - 7, T - 3], 3, 4, 1, "fp32", True, False, True, True)
    _check((T,), [10, T], 3, 4, 1, "fp32", True, False, False, False)


def _fixed(T=300, H=40, N=16, dtype=torch.float32, seed=4):
    g = torch.Generator().manual_seed(seed)
    t = {"x": torch.randn(2, T, H, generator=g).to(dtype), "delta": torch.randn(2, T, H, generator=g).to(dtype) * 0.5,
         "A": -torch.rand(H, N, generator=g) * 4, "B": torch.randn(2, T, N, generator=g).to(dtype),
         "C": torch.randn(2, T, N, generator=g).to(dtype), "D": torch.randn(H, generator=g),
         "z": torch.randn(2, T, H, generator=g).to(dtype), "delta_bias": torch.randn(H, generator=g) - 2,
         "state": torch.randn(2, H, N, generator=g)}
    return {k: v.to(DEV) for k, v in t.items()}


def test_same_bits_any_stream_any_layout():
    t = _fixed()
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}

    def run(kw):
        o, h = ltc_cuda.ltc_selective_scan(**kw, delta_softplus=True)
        return [o, h, *torch.autograd.grad([o, h], list(leaves.values()), [torch.ones_like(o), h.detach()])]

    first = run(leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(leaves)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    # projections cut out of one tensor, time first, and channels that are not last
    both = torch.cat([t["B"], t["C"]], -1)
    views = dict(t, B=both[..., :16], C=both[..., 16:], x=t["x"].transpose(0, 1).contiguous().transpose(0, 1),
                 z=t["z"].transpose(1, 2).contiguous().transpose(1, 2))
    o, h = ltc_cuda.ltc_selective_scan(**views, delta_softplus=True)
    assert torch.equal(o, first[0]) and torch.equal(h, first[1])
    part = dict(t, x=torch.cat([t["x"], t["x"]], -1)[..., :40], delta=t["delta"].repeat(1, 2, 1)[:, ::2][:, :300])
    want = dict(part, x=part["x"].contiguous(), delta=part["delta"].contiguous())
    # step sizes taken as they are: the negative ones here let states grow to NaN
    a, b = ltc_cuda.ltc_selective_scan(**part)[0], ltc_cuda.ltc_selective_scan(**want)[0]
    assert bool(((a == b) | (a.isnan() & b.isnan())).all())


def test_pieces_are_the_whole():
    """A sequence in two calls, the state handed on, is the sequence in one: off by the
    roundings of its chunks, which are cut elsewhere."""
    t = _fixed(T=200)
    seq = ("x", "delta", "B", "C", "z")
    o, h = ltc_cuda.ltc_selective_scan(**t, delta_softplus=True)
    a = {k: v[:, :77] if k in seq else v for k, v in t.items()}
    b = {k: v[:, 77:] if k in seq else v for k, v in t.items()}
    oa, ha = ltc_cuda.ltc_selective_scan(**a, delta_softplus=True)
    ob, hb = ltc_cuda.ltc_selective_scan(**dict(b, state=ha), delta_softplus=True)
    size = o.abs().max()
    assert float((torch.cat([oa, ob], 1) - o).abs().max() / size) <= 40 * 200 * U
    assert float((hb - h).abs().max() / h.abs().max()) <= 40 * 200 * U


def test_gradients_of_one_output_or_input():
    t = _fixed(T=90)
    for k in t:
        leaf = t[k].clone().requires_grad_(True)
        o, h = ltc_cuda.ltc_selective_scan(**dict(t, **{k: leaf}), delta_softplus=True)
        alone, = torch.autograd.grad(o, [leaf], torch.ones_like(o))
        every = {n: v.clone().requires_grad_(True) for n, v in t.items()}
        o, h = ltc_cuda.ltc_selective_scan(**every, delta_softplus=True)
        assert torch.equal(alone, torch.autograd.grad(o.sum(), [every[k]])[0]), k
    every = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    o, h = ltc_cuda.ltc_selective_scan(**every, delta_softplus=True)
    g = torch.autograd.grad(h.sum(), [every["C"], every["x"], every["state"]], allow_unused=True)
    assert float(g[0].abs().max()) == 0 and float(g[1].abs().max()) > 0
    # an input that two leaves share
    both = t["B"].clone().requires_grad_(True)
    o, h = ltc_cuda.ltc_selective_scan(**dict(t, B=both, C=both), delta_softplus=True)
    s, = torch.autograd.grad(o.sum(), [both])
    o, h = ltc_cuda.ltc_selective_scan(**dict(every, C=every["C"], B=every["B"]), delta_softplus=True)
    b = t["B"].clone().requires_grad_(True)
    c = t["B"].clone().requires_grad_(True)
    o, h = ltc_cuda.ltc_selective_scan(**dict(t, B=b, C=c), delta_softplus=True)
    assert torch.equal(s, sum(torch.autograd.grad(o.sum(), [b, c])))


@pytest.mark.parametrize("where", ["x", "delta", "B", "C", "z"])
def test_what_lies_outside_stays_there(where):
    """NaN and infinities before the first sequence, behind the last and in another."""
    g = torch.Generator().manual_seed(1)
    T, H, N = 90, 20, 16
    cu = torch.tensor([3, 40, 41, 75], dtype=torch.int32, device=DEV)
    t = {"x": torch.randn(T, H, generator=g), "delta": torch.rand(T, H, generator=g),
         "B": torch.randn(T, N, generator=g), "C": torch.randn(T, N, generator=g),
         "z": torch.randn(T, H, generator=g)}
    t = {k: v.to(DEV) for k, v in t.items()}
    A = -torch.rand(H, N, device=DEV)

    def run(kw, leaf=False):
        kw = {k: v.clone().requires_grad_(leaf) for k, v in kw.items()}
        o, h = ltc_cuda.ltc_selective_scan(**kw, A=A, cu_seqlens=cu)
        if not leaf:
            return o, h
        return o, h, dict(zip(kw, torch.autograd.grad(o, list(kw.values()), torch.ones_like(o))))

    o, h, grads = run(t, True)
    bad = {k: v.clone() for k, v in t.items()}
    bad[where][:3] = float("nan")
    bad[where][75:] = float("inf")
    o2, h2, grads2 = run(bad, True)
    assert torch.equal(o, o2) and torch.equal(h, h2)
    for k in grads:
        assert torch.equal(grads[k], grads2[k]), k
        assert float(grads2[k][75:].abs().max()) == 0 and float(grads2[k][:3].abs().max()) == 0
    bad[where][40] = float("nan")  # the second sequence, one token
    o3, h3, grads3 = run(bad, True)
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[40] = False
    assert torch.equal(o[keep], o3[keep]) and torch.equal(h[[0, 2]], h3[[0, 2]])
    for k in grads:
        assert torch.equal(grads[k][keep], grads3[k][keep]), k


def test_large_steps_and_values():
    """Steps whose decays vanish, softplus far on both sides, and an infinite input."""
    t = _fixed(T=40, N=4)
    t["delta"][:, 10] = 80.0
    t["delta"][:, 11] = -80.0
    d = {k: v.cpu().double() for k, v in t.items()}
    want, hf = R.scan(d["x"], d["delta"], d["A"], d["B"][:, :, None], d["C"][:, :, None], d["D"], d["z"],
                      d["delta_bias"], d["state"], None, True)
    o, h = ltc_cuda.ltc_selective_scan(**t, delta_softplus=True)
    assert float((o.cpu().double() - want).abs().max() / want.abs().max()) <= 40 * 40 * U
    t["x"][0, 20, 3] = float("inf")
    o2, _ = ltc_cuda.ltc_selective_scan(**t, delta_softplus=True)
    same = torch.ones_like(o, dtype=torch.bool)
    same[0, 20:, 3] = False
    assert torch.equal(o[same], o2[same]) and not bool(o2[0, 20, 3].isfinite())


def test_gradient_by_differences():
    """A directional derivative over all inputs: central differences are off by h^2 / 6 of
    the third one and by the outputs' roundings over h, below 2e-3 of the size here."""
    t = {k: v.requires_grad_(True) for k, v in _fixed(T=40, H=6, N=5).items()}
    c = torch.randn(2, 40, 6, device=DEV)

    def loss(kw):
        o, h = ltc_cuda.ltc_selective_scan(**kw, delta_softplus=True)
        return (o.double() * c).sum() + h.double().sum()

    grads = torch.autograd.grad(loss(t), list(t.values()))
    dirs = [torch.randn_like(v) for v in t.values()]
    h = 2.0 ** -8
    with torch.no_grad():
        up, down = (loss({k: v + s * h * e for (k, v), e in zip(t.items(), dirs)}) for s in (1, -1))
    num = (up - down) / (2 * h)
    ana = sum((g.double() * e).sum() for g, e in zip(grads, dirs))
    size = sum((g.double() * e).abs().sum() for g, e in zip(grads, dirs))
    assert abs(float(num - ana)) <= 2e-3 * float(size)


@pytest.mark.parametrize("B,H,N,G,dtype,skip,gated,softplus,pool", [
    (1, 4, 16, 1, "fp32", True, True, True, 0), (4, 70, 16, 1, "bf16", True, True, True, 9),
    (5, 12, 5, 3, "fp32", False, False, False, 5), (6, 33, 64, 1, "fp16", True, False, True, 8),
    (4, 130, 1, 2, "fp32", True, True, True, 6), (0, 8, 4, 1, "fp32", True, True, True, 2)])
def test_step(B, H, N, G, dtype, skip, gated, softplus, pool):
    """Steps are the scan token by token: padding, absent and repeated slots too."""
    P = pool or B
    slots = None
    if pool:
        slots = torch.arange(B, dtype=torch.int32) % P
        if B > 3:
            slots[1], slots[2], slots[3] = -1, slots[0], P
    state = torch.randn(P, H, N, generator=torch.Generator().manual_seed(8))
    held, state = state.double(), state.to(DEV)
    for k in range(3):
        t = _inputs((max(B, 1),), 0, H, N, G, dtype, skip, gated, softplus, False, seed=k)
        t = {n: v if v is None or n in ("A", "D", "bias") else v[:B] for n, v in t.items()}
        d = {n: None if v is None else v.to(DEV) for n, v in t.items()}
        bm, cm = (d[n].squeeze(-2) if G == 1 else d[n] for n in "BC")
        out = ltc_cuda.ltc_selective_scan_step(d["x"], d["delta"], d["A"], bm, cm, state, d["D"], d["z"],
                                               d["bias"], None if slots is None else slots.to(DEV), softplus)
        assert out.shape == (B, H) and out.dtype == R.TYPES[dtype]
        for r in range(B):
            at = r if slots is None else int(slots[r])
            if at < 0:
                assert float(out[r].abs().max()) == 0
                continue
            if at >= P:
                assert bool(out[r].isnan().all())
                continue
            one = {n: None if v is None else v.double() if n in ("A", "D", "bias") else v[r].double()[None, None]
                   for n, v in t.items()}
            one["state"] = held[at][None]
            y, h = R.scan(one["x"], one["delta"], one["A"], one["B"], one["C"], one["D"], one["z"],
                          one["bias"], one["state"], None, softplus)
            zero = torch.zeros_like(one["x"])
            mo, mh, _ = _sizes(one, None, softplus, zero, torch.zeros_like(one["state"]))
            _close(out[r], y[0, 0], mo[0, 0], dtype, 3 * 40 + 16 + N, "out")
            held[at] = h[0]
            _close(state[at], h[0], mh[0], "fp32", 3 * 40, "state") if slots is None else None
    if B:
        live = range(P) if slots is None else {int(s) for s in slots if 0 <= s < P}
        for at in live:
            assert float((state[at].cpu().double() - held[at]).abs().max()) <= 200 * U * (
                1 + float(held[at].abs().max()))


def test_step_strided_state():
    big = torch.randn(6, 2, 8, 16, device=DEV)
    keep = big.clone()
    state, dense = big[:, 0], big[:, 0].contiguous()
    t = {k: v.to(DEV) for k, v in _inputs((6,), 0, 8, 16, 1, "fp32", True, True, True, False).items()
         if v is not None}
    args = (t["x"], t["delta"], t["A"], t["B"].squeeze(-2), t["C"].squeeze(-2))
    a = ltc_cuda.ltc_selective_scan_step(*args, dense, t["D"], t["z"], t["bias"], None, True)
    b = ltc_cuda.ltc_selective_scan_step(*args, state, t["D"], t["z"], t["bias"], None, True)
    assert torch.equal(a, b) and torch.equal(state, dense) and torch.equal(big[:, 1], keep[:, 1])


def test_refusals():
    t = _fixed(T=5, H=8, N=4)
    f = ltc_cuda.ltc_selective_scan

    def wrong(exc, **kw):
        with pytest.raises(exc):
            f(**dict(t, **kw))

    wrong(ValueError, A=t["A"].cpu())
    wrong(ValueError, x=t["x"].cpu())
    wrong(TypeError, x=t["x"].double())
    wrong(TypeError, delta=t["delta"].half())
    wrong(ValueError, delta=t["delta"][:, :4])
    wrong(TypeError, A=t["A"].double())
    wrong(ValueError, A=t["A"][:7])
    wrong(ValueError, A=torch.zeros(8, 65, device=DEV), B=torch.zeros(2, 5, 65, device=DEV),
          C=torch.zeros(2, 5, 65, device=DEV), state=None)
    wrong(ValueError, B=t["B"][..., :3])
    wrong(ValueError, C=t["C"][:, :, None])
    wrong(ValueError, B=t["B"][:, :, None].repeat(1, 1, 3, 1), C=t["C"][:, :, None].repeat(1, 1, 3, 1))
    wrong(TypeError, B=t["B"].half())
    wrong(ValueError, D=t["D"][:7])
    wrong(TypeError, D=t["D"].half())
    wrong(TypeError, z=t["z"].half())
    wrong(ValueError, state=t["state"][:1])
    wrong(TypeError, state=t["state"].half())
    wrong(ValueError, delta_bias=t["delta_bias"][:3])
    wrong(ValueError, cu_seqlens=torch.tensor([0, 5], dtype=torch.int32, device=DEV))
    s = ltc_cuda.ltc_selective_scan_step
    one = {k: v[:, 0] if k in ("x", "delta", "B", "C", "z") else v for k, v in t.items()}
    s(**one)
    for exc, kw in ((ValueError, {"state": t["state"][:1]}), (TypeError, {"state": t["state"].half()}),
                    (ValueError, {"state": t["state"][:1].expand(2, 8, 4)}),
                    (ValueError, {"state": t["state"].transpose(1, 2).contiguous().transpose(1, 2)}),
                    (ValueError, {"x": t["state"][:, :, 0]}),
                    (RuntimeError, {"x": one["x"].clone().requires_grad_(True)})):
        with pytest.raises(exc):
            s(**dict(one, **kw))
