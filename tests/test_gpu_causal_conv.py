"""The causal convolution against its definition in 64 bits: lengths from none to several
runs, packed and strided, with and without a state; its gradients, and its step.

Tolerances count roundings. A sum of K products and a bias is K + 1 multiply-adds, each off
by at most half a step of 2^-24 of the sum of the terms' sizes; silu adds an exponential
(whose argument's rounding counts |v| of them, at most 8 here), a sum, a reciprocal and a
product. So an output is off by at most 2^-24 (K + 16) times the sum of the sizes, and by
half a step of its own type. The slope of silu in a gradient has two more products."""

from __future__ import annotations

import pytest
import torch

import _model_ref as R
import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _inputs(shape, K, dtype, wtype, bias, state, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g).to(R.TYPES[dtype])
    C = shape[-1]
    w = (torch.rand(C, K, generator=g) * 2 - 1).to(R.TYPES[wtype])
    b = (torch.randn(C, generator=g) * 0.3).to(R.TYPES[wtype]) if bias else None
    s = torch.randn(rows, K - 1, C, generator=g).to(R.TYPES[dtype]) if state else None
    return x, w, b, s


def _dev(t, grad=False):
    return None if t is None else t.to(DEV).requires_grad_(grad)


def _dbl(t, grad=False):
    return None if t is None else t.double().requires_grad_(grad)


def _close(got, want, mag, dtype, count):
    got, want = got.detach().cpu().double(), want.detach()
    tol = R.half_step(dtype) * (want.abs() + count * U * mag) + count * U * mag
    tol = tol + torch.finfo(R.TYPES[dtype]).tiny
    off = (got - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), float((off / tol).max())


def _sizes(x, w, b, s, cu):
    return R.conv(x.double().abs(), w.double().abs(), None if b is None else b.double().abs(),
                  None if s is None else s.double().abs(), cu)[0]


SHAPES = [((2, 1, 4), None), ((3, 2, 8), None), ((2, 9, 40), None), ((1, 70, 130), None),
          ((2, 131, 17), None), ((5, 0, 8), None), ((0, 5, 8), None), ((1, 300, 1), None),
          ((40, 24), [0, 3, 3, 4, 30, 36]), ((200, 33), [2, 2, 9, 140, 141, 190]),
          ((7, 8), [0, 7]), ((9, 8), [9, 9]), ((6, 16), [0, 0, 0]), ((5, 8), [3])]


@pytest.mark.parametrize("shape,cu", SHAPES)
@pytest.mark.parametrize("K,dtype,wtype,bias,state,act", [
    (4, "fp32", "fp32", True, True, "silu"), (4, "bf16", "bf16", True, False, "silu"),
    (3, "fp16", "fp32", False, True, None), (1, "bf16", "fp32", True, False, "silu"),
    (2, "fp32", "fp32", False, False, None), (8, "bf16", "bf16", True, True, "silu"),
    (5, "fp16", "fp16", True, True, "silu"), (7, "fp32", "fp32", True, True, None),
    (6, "bf16", "fp32", False, True, "silu")])
def test_forward_and_gradients(shape, cu, K, dtype, wtype, bias, state, act):
    rows = shape[0] if cu is None else len(cu) - 1
    x, w, b, s = _inputs(shape, K, dtype, wtype, bias, state, rows)
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    xd, wd, bd, sd = (_dbl(t, True) for t in (x, w, b, s))
    want, tail = R.conv(xd, wd, bd, sd, c, act)
    xg, wg, bg, sg = (_dev(t, True) for t in (x, w, b, s))
    out, hf = ltc_cuda.ltc_causal_conv(xg, wg, bg, sg, None if c is None else c.to(DEV), act)
    assert out.dtype == xg.dtype and hf.shape == (rows, K - 1, shape[-1])
    mag = _sizes(x, w, b, s, c)
    _close(out, want, mag, dtype, K + 16)
    assert torch.equal(hf.detach().cpu().double(), tail.detach())
    g = torch.Generator().manual_seed(5)
    go = torch.randn(shape, generator=g).to(x.dtype)
    gh = torch.randn(hf.shape, generator=g).to(x.dtype)
    leaves = [(n, a, d) for n, a, d in (("x", xg, xd), ("w", wg, wd), ("b", bg, bd), ("s", sg, sd))
              if a is not None]
    got = torch.autograd.grad([out, hf], [a for _, a, _ in leaves], [go.to(DEV), gh.to(DEV)])
    ref = R.gradients([want, tail], [go.double(), gh.double()], [d for _, _, d in leaves])
    # sizes of the terms: the same sums of sizes, a slope of at most 1.1
    absd = [None if t is None else t.double().abs().requires_grad_(True) for t in (x, w, b, s)]
    o, h = R.conv(*absd, c, None)
    by = dict(zip("xwbs", absd))
    sizes = R.gradients([o, h], [go.double().abs() * 1.1, gh.double().abs()],
                        [by[n] for n, _, _ in leaves])
    # a slope is off by as much as the pre-activation is, and by 24 roundings of its own;
    # sums over tokens add one a token, in at most 16 parts each
    tokens = x.numel() // max(1, shape[-1])
    for (n, _, _), a, r, m in zip(leaves, got, ref, sizes):
        grow = float(mag.max()) if mag.numel() else 0.0
        count = K + 24 + (K + 4) * grow + (tokens + 16 if n in "wb" else K)
        kind = dtype if n in "xs" else wtype
        _close(a, r, m, kind, count)


def test_strides_streams_and_order():
    """Views of other layouts, another stream, and the same bits in every call."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(4, 50, 3, 24, generator=g).to(DEV)
    w = torch.randn(24, 4, generator=g).to(DEV)
    for v in (base[:, :, 1], base[1:, ::2, 0, :], base[:, :, 2].transpose(0, 1), base.transpose(2, 3)[:, :, :, 0]):
        a = ltc_cuda.ltc_causal_conv(v, w, activation="silu")[0]
        b = ltc_cuda.ltc_causal_conv(v.contiguous(), w, activation="silu")[0]
        assert torch.equal(a, b)
    x = base[:, :, 1].contiguous().requires_grad_(True)
    w.requires_grad_(True)

    def run():
        o, h = ltc_cuda.ltc_causal_conv(x, w, activation="silu")
        return [o, h, *torch.autograd.grad([o, h], [x, w], [torch.ones_like(o), torch.ones_like(h)])]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    # an expanded gradient, and none for one of the outputs
    o, h = ltc_cuda.ltc_causal_conv(x, w, activation="silu")
    ones = torch.autograd.grad(o.sum(), [x, w])
    o, h = ltc_cuda.ltc_causal_conv(x, w, activation="silu")
    dense = torch.autograd.grad(o, [x, w], torch.ones_like(o))
    assert all(torch.equal(a, b) for a, b in zip(ones, dense))
    o, h = ltc_cuda.ltc_causal_conv(x, w)
    gx, = torch.autograd.grad(h.sum(), [x])
    assert float(gx[:, :-3].abs().max()) == 0 and torch.equal(gx[:, -3:], torch.ones_like(gx[:, -3:]))


def test_what_lies_outside_stays_there():
    """NaN behind the last sequence, in another sequence and in other channels."""
    x = torch.randn(40, 16, device=DEV)
    cu = torch.tensor([2, 20, 33], dtype=torch.int32, device=DEV)
    w = torch.randn(16, 4, device=DEV)
    clean = ltc_cuda.ltc_causal_conv(x, w, cu_seqlens=cu)
    bad = x.clone()
    bad[33:] = float("nan")
    bad[:2] = float("inf")
    bad[19, 3] = float("nan")
    leaf = bad.clone().requires_grad_(True)
    out, hf = ltc_cuda.ltc_causal_conv(leaf, w, cu_seqlens=cu)
    gx, = torch.autograd.grad(out, [leaf], torch.ones_like(out))
    same = torch.ones(40, 16, dtype=torch.bool, device=DEV)
    same[19, 3] = False
    assert torch.equal(out[same], clean[0][same]) and bool(out[19, 3].isnan())
    assert float(out[33:].abs().max()) == 0 and float(out[:2].abs().max()) == 0
    assert float(gx[33:].abs().max()) == 0 and bool(gx.isfinite().all())


@pytest.mark.parametrize("B,C,K,dtype,wtype,act,pool", [
    (1, 4, 4, "fp32", "fp32", "silu", 0), (3, 130, 4, "bf16", "fp32", "silu", 7),
    (9, 33, 2, "fp16", "fp16", None, 12), (4, 700, 8, "bf16", "bf16", "silu", 4),
    (5, 16, 1, "fp32", "fp32", "silu", 6), (0, 8, 4, "fp32", "fp32", None, 3)])
def test_step(B, C, K, dtype, wtype, act, pool):
    """Steps are the convolution token by token: padding, absent and repeated slots too."""
    P = pool or B
    x, w, b, s = _inputs((3, max(B, 1), C), K, dtype, wtype, True, True, max(P, 1), seed=2)
    x, s = x[:, :B], s[:P]
    wd, bd = w.double(), b.double()
    slots = None
    if pool:
        slots = torch.arange(B, dtype=torch.int32) % P
        if B > 2:
            slots[1], slots[2] = -1, slots[0]
        if B > 3:
            slots[3] = P
    state = s.to(DEV)
    held = s.double()
    for t in range(3):
        out = ltc_cuda.ltc_causal_conv_step(x[t].to(DEV), w.to(DEV), state, b.to(DEV),
                                            None if slots is None else slots.to(DEV), act)
        for r in range(B):
            k = r if slots is None else int(slots[r])
            if k < 0:
                assert float(out[r].abs().max()) == 0
                continue
            if k >= P:
                assert bool(out[r].isnan().all())
                continue
            y, tail = R.conv(x[t, r].double()[None, None], wd, bd, held[k][None], None, act)
            mag = _sizes(x[t, r][None, None], w, b, held[k][None], None)
            _close(out[r], y[0, 0], mag[0, 0], dtype, K + 16)
            held[k] = tail[0]
        assert torch.equal(state.cpu().double(), held)


def test_step_strided_state():
    """A pool whose rows lie apart is updated where it is, and nothing between them."""
    big = torch.randn(5, 4, 40, device=DEV)
    keep = big.clone()
    state = big[:, :3, :32]
    x, w = torch.randn(5, 32, device=DEV), torch.randn(32, 4, device=DEV)
    dense = state.contiguous()
    a = ltc_cuda.ltc_causal_conv_step(x, w, dense)
    b = ltc_cuda.ltc_causal_conv_step(x, w, state)
    assert torch.equal(a, b) and torch.equal(state, dense)
    assert torch.equal(big[:, 3], keep[:, 3]) and torch.equal(big[:, :, 32:], keep[:, :, 32:])


def test_gradient_by_differences():
    """A directional derivative: central differences are off by h^2 / 6 of the third one,
    and by the outputs' roundings over h; both are below 2e-3 of the size here."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 30, 12, generator=g).to(DEV).requires_grad_(True)
    w = torch.randn(12, 4, generator=g).to(DEV).requires_grad_(True)
    c = torch.randn(2, 30, 12, generator=g).to(DEV)

    def loss(a, b):
        return (ltc_cuda.ltc_causal_conv(a, b, activation="silu")[0].double() * c).sum()

    gx, gw = torch.autograd.grad(loss(x, w), [x, w])
    dx, dw = torch.randn_like(x), torch.randn_like(w)
    h = 2.0 ** -7
    with torch.no_grad():
        num = (loss(x + h * dx, w + h * dw) - loss(x - h * dx, w - h * dw)) / (2 * h)
    ana = (gx.double() * dx).sum() + (gw.double() * dw).sum()
    size = (gx.double() * dx).abs().sum() + (gw.double() * dw).abs().sum()
    assert abs(float(num - ana)) <= 2e-3 * float(size)


def test_refusals():
    x, w = torch.randn(2, 5, 8, device=DEV), torch.randn(8, 4, device=DEV)
    f = ltc_cuda.ltc_causal_conv
    for bad, exc in ((lambda: f(x.cpu(), w.cpu()), ValueError), (lambda: f(x, w.cpu()), ValueError),
                     (lambda: f(x.double(), w), TypeError), (lambda: f(x, w.bfloat16()), TypeError),
                     (lambda: f(x, w[:7]), ValueError), (lambda: f(x[0], w), ValueError),
                     (lambda: f(x, torch.randn(8, 9, device=DEV)), ValueError),
                     (lambda: f(x, torch.randn(8, 0, device=DEV)), ValueError),
                     (lambda: f(x, w, torch.randn(7, device=DEV)), ValueError),
                     (lambda: f(x, w, torch.randn(8, device=DEV).half()), TypeError),
                     (lambda: f(x, w, state=torch.randn(2, 4, 8, device=DEV)), ValueError),
                     (lambda: f(x, w, state=torch.randn(2, 3, 8, device=DEV).half()), TypeError),
                     (lambda: f(x, w, activation="tanh"), ValueError),
                     (lambda: f(x[0], w, cu_seqlens=torch.tensor([0, 5], device=DEV)), TypeError)):
        with pytest.raises(exc):
            bad()
    st = torch.randn(2, 3, 8, device=DEV)
    s = ltc_cuda.ltc_causal_conv_step
    xs = torch.randn(2, 8, device=DEV)
    for bad, exc in ((lambda: s(xs, w, st[:1]), ValueError), (lambda: s(xs, w, st.half()), TypeError),
                     (lambda: s(xs, w, st[:1].expand(2, 3, 8)), ValueError),
                     (lambda: s(xs, w, st.transpose(0, 1)[:, :2]), ValueError),
                     (lambda: s(st[0, :2], w, st), ValueError),
                     (lambda: s(xs, w, st, slots=torch.zeros(2, device=DEV, dtype=torch.int64)), TypeError),
                     (lambda: s(xs.requires_grad_(True), w, st), RuntimeError)):
        with pytest.raises(exc):
            bad()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(f(leaf, w)[0].sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()
