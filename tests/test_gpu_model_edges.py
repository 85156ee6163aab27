"""The convolution and the selective scan where their inputs are at an edge of what is
allowed: boundaries of packed sequences in any order, channels that are not finite,
states that grow, sums over many tokens."""

from __future__ import annotations

import pytest
import torch

import _model_ref as R
import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"

ODD_BOUNDARIES = [[0, 40, 20, 64], [-5, 10, 64], [0, 10, 1000], [70, 80, 90], [64, 0], [2 ** 31 - 1, -2 ** 31],
                  [0, 10, 3, 0], [3, 1, -3], [0, 33, 17, 0, 0], [50, 64, 5, 64, 0, 70]]


@pytest.mark.parametrize("cu", ODD_BOUNDARIES)
@pytest.mark.parametrize("T,N", [(64, 4), (200, 24)])
def test_boundaries_out_of_order_or_range_stay_in_bounds(cu, T, N):
    """Unspecified results, but no access out of range: whole calls, and a C call whose
    states lie between others."""
    g = torch.Generator().manual_seed(1)
    c = torch.tensor(cu, dtype=torch.int32, device=DEV)
    S, H = len(cu) - 1, 6

    def leaf(*shape):
        return torch.randn(*shape, generator=g).to(DEV).requires_grad_(True)

    x, w, b, tail = leaf(T, H), leaf(H, 4), leaf(H), leaf(S, 3, H)
    out, hf = ltc_cuda.ltc_causal_conv(x, w, b, tail, c, "silu")
    grads = torch.autograd.grad([out, hf], [x, w, b, tail], [torch.ones_like(out), torch.ones_like(hf)])
    assert out.shape == x.shape and hf.shape == tail.shape and grads[3].shape == tail.shape
    delta, B, C, state = leaf(T, H), leaf(T, N), leaf(T, N), leaf(S, H, N)
    A = (-torch.rand(H, N, generator=g)).to(DEV).requires_grad_(True)
    leaves = [x, delta, A, B, C, state]
    out, hf = ltc_cuda.ltc_selective_scan(x, delta, A, B, C, state=state, cu_seqlens=c, delta_softplus=True)
    grads = torch.autograd.grad([out, hf], leaves, [torch.ones_like(out), torch.ones_like(hf)])
    assert out.shape == x.shape and hf.shape == state.shape and grads[5].shape == state.shape
    # final states and the initial ones' gradients between 64 rows of others
    lib = ltc_cuda._cuda_module.capi.lib
    sizes = (S, T, H, N, 1, 1)
    row = H * N
    around = torch.full((2, S + 128, row), 7.0, device=DEV)
    ends = [around[k, 64:64 + S].data_ptr() for k in range(2)]
    o, saved = torch.empty(T, H, device=DEV), torch.empty(lib.ltc_selective_scan_saved_floats(*sizes), device=DEV)
    need = max(lib.ltc_selective_scan_fwd_workspace_bytes(*sizes), lib.ltc_selective_scan_bwd_workspace_bytes(*sizes))
    ws = torch.empty(need + 256, dtype=torch.uint8, device=DEV)
    at = (ws.data_ptr() + 255) // 256 * 256
    ins = (x.data_ptr(), 0, H, delta.data_ptr(), 0, H, A.data_ptr(), B.data_ptr(), 0, N, 0, C.data_ptr(), 0, N, 0,
           None, None, 0, 0, None, state.data_ptr(), c.data_ptr(), 0, 1, S, T, H, N, 1)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ltc_selective_scan_forward(*ins, 1, o.data_ptr(), ends[0], saved.data_ptr(), at, need, stream) == 0
    ones, gh = torch.ones(T, H, device=DEV), torch.ones(S, H, N, device=DEV)
    assert lib.ltc_selective_scan_backward(*ins, saved.data_ptr(), ones.data_ptr(), 0, H, gh.data_ptr(), None, None,
                                           None, None, None, None, None, None, ends[1], at, need, stream) == 0
    torch.cuda.synchronize()
    assert bool((around[:, :64] == 7).all()) and bool((around[:, 64 + S:] == 7).all())


@pytest.mark.parametrize("H,G,N,dtype", [(10, 2, 16, "fp32"), (10, 2, 24, "bf16"), (140, 2, 5, "fp32"),
                                         (195, 3, 40, "fp16")])
@pytest.mark.parametrize("T,cu", [(40, None), (200, None), (200, [0, 30, 190])])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_channel_that_is_not_finite_stays_in_its_group(H, G, N, dtype, T, cu, bad):
    """Groups that do not fill blocks of 64 channels: the first channel's state and inputs
    are in the gradients of its own group's B and C, and in no other's."""
    g = torch.Generator().manual_seed(2)
    dt, lead = R.TYPES[dtype], (T,) if cu else (1, T)
    rows = len(cu) - 1 if cu else 1

    def rand(*shape, t=dt):
        return torch.randn(*shape, generator=g).to(t).to(DEV)

    t = {"x": rand(*lead, H), "delta": rand(*lead, H), "A": -rand(H, N, t=torch.float32).abs(),
         "B": rand(*lead, G, N), "C": rand(*lead, G, N), "D": rand(H, t=torch.float32), "z": rand(*lead, H),
         "state": rand(rows, H, N, t=torch.float32)}
    go, gh = rand(*lead, H), rand(rows, H, N, t=torch.float32)
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)

    def run(kw):
        kw = {k: v.clone().requires_grad_(True) for k, v in kw.items()}
        out, hf = ltc_cuda.ltc_selective_scan(**kw, cu_seqlens=c, delta_softplus=True)
        return out, hf, dict(zip(kw, torch.autograd.grad([out, hf], list(kw.values()), [go, gh])))

    out, hf, grads = run(t)
    for name in ("state", "x"):
        kw = {k: v.clone() for k, v in t.items()}
        if name == "state":
            kw["state"][:, 0] = bad
        else:
            kw["x"][..., 0] = bad
        o, h, got = run(kw)
        assert not bool(o[..., 0].isfinite().all())
        assert torch.equal(o[..., 1:], out[..., 1:]) and torch.equal(h[:, 1:], hf[:, 1:])
        for k in ("B", "C"):
            assert torch.equal(got[k][..., 1:, :], grads[k][..., 1:, :]), (name, k)
        for k in ("x", "delta", "z"):
            assert torch.equal(got[k][..., 1:], grads[k][..., 1:]), (name, k)
        assert torch.equal(got["A"][1:], grads["A"][1:]) and torch.equal(got["D"][1:], grads["D"][1:])
        assert torch.equal(got["state"][:, 1:], grads["state"][:, 1:])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_states_that_grow_past_a_chunk(dtype):
    """Decays above 1 whose product over a chunk is past float32's range: a state of zero
    stays zero, a small one grows to what it is by definition, and so backward."""
    dt = R.TYPES[dtype]
    T, H, N = 200, 3, 4
    one = torch.ones(1, T, H)
    t = {"x": torch.zeros(1, T, H), "delta": one.clone(), "A": torch.full((H, N), 2.0),
         "B": torch.ones(1, T, N), "C": torch.ones(1, T, N)}
    t["x"][:, -5:] = 0.5

    def dev(kw):
        return {k: v.to(DEV, v.dtype if k in ("A", "state") else dt).requires_grad_(True) for k, v in kw.items()}

    def run(kw, state=None, go=None, gh=None):
        kw = dev(kw if state is None else dict(kw, state=state))
        out, hf = ltc_cuda.ltc_selective_scan(**kw)
        if go is None and gh is None:
            return out.detach().cpu().double(), hf.detach().cpu().double()
        outs, grads = ([out], [go.to(DEV, dt)]) if gh is None else ([hf], [gh.to(DEV)])
        return dict(zip(kw, torch.autograd.grad(outs, list(kw.values()), grads, allow_unused=True)))

    def definition(kw, state=None):
        d = {k: v.double() for k, v in kw.items()}
        return R.scan(d["x"], d["delta"], d["A"], d["B"][:, :, None], d["C"][:, :, None],
                      state=None if state is None else state.double())

    def close(got, want, steps):
        # a token's exponent of 3 at most, and its other roundings: 40 a token
        tol = (40 * steps * 2.0 ** -24 + (R.half_step(dtype) if got.dtype == dt else 0)) * want.abs()
        return bool(((got.detach().cpu().double() - want).abs() <= tol).all())

    out, hf = run(t)
    want, whf = definition(t)
    assert float(out[:, :-5].abs().max()) == 0 and bool(out.isfinite().all())
    tol = (40 * 5 * 2.0 ** -24 + R.half_step(dtype)) * want.abs()
    assert bool(((out - want).abs() <= tol).all()) and close(hf, whf, 5)
    # a state of 1e-30 that grows by e^150 in 100 tokens, the first 64 of which are a chunk
    small = {k: v[:, :100] if k != "A" else v for k, v in t.items()}
    small["x"], small["delta"], small["A"] = torch.zeros(1, 100, H), one[:, :100] * 1.5, torch.ones(H, N)
    state = torch.full((1, H, N), 1e-30)
    _, hf = run(small, state)
    assert close(hf, definition(small, state)[1], 100)
    # backward: a gradient of the first tokens alone, and one of 1e-30 that grows
    none = dict(t, x=torch.zeros(1, T, H))
    go = torch.zeros(1, T, H)
    go[:, :5] = 1.0
    got = run(none, go=go)
    gx = torch.zeros(T)
    for i in range(5):
        gx[i] = sum(2.718281828459045 ** (2.0 * (j - i)) for j in range(i, 5)) * N
    assert close(got["x"], gx.double().view(1, T, 1).expand(1, T, H), 5 + 8)
    assert all(bool(v.isfinite().all()) for v in got.values())
    got = run(small, torch.zeros(1, H, N), gh=torch.full((1, H, N), 1e-30))
    assert close(got["state"], torch.full((1, H, N), 2.718281828459045 ** 150 * float(torch.tensor(1e-30))).double(), 100)


@pytest.mark.parametrize("B,T,cu", [(256, 32768, None), (4096, 16, None), (3, 5, None), (1, 70000, None),
                                    (0, 300000, [0, 100000, 100001, 299999]), (0, 40, [3, 40])])
def test_sums_over_tokens_do_not_lose_with_their_number(B, T, cu):
    """The gradients of A, D and the bias add a term a token. Decays of 1 and states of 1
    make every other operation exact, and every term 1.3: each sum is off by its roundings
    alone. In units of 2^-24: a batch of 16 tokens 15, the running sum, which carries its
    error along, 2, eight waves 7 (D and the bias), the blocks 2 and their eight parts 7:
    33 at most, however many tokens."""
    n = B * T if cu is None else cu[-1] - cu[0]
    lead, rows = ((B, T), B) if cu is None else ((T,), len(cu) - 1)
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
    term = torch.tensor(1.3)

    def full(v, *shape):
        return torch.full(shape, float(v), device=DEV)

    zero, one = full(0, *lead, 1), full(1, *lead, 1)
    state, gh = full(1, rows, 1, 1), full(1, rows, 1, 1)
    want = n * float(term.double())

    def off(x, delta):
        leaves = {"A": full(0, 1, 1), "D": full(0, 1), "delta_bias": full(0, 1)}
        leaves = {k: v.requires_grad_(True) for k, v in leaves.items()}
        out, hf = ltc_cuda.ltc_selective_scan(x, delta, B=one, C=zero, state=state, cu_seqlens=c, **leaves)
        got = torch.autograd.grad([out, hf], list(leaves.values()), [one, gh])
        return [abs(float(v.double()) - want) / want / 2.0 ** -24 for v in got]

    errors = [off(zero, one * term.to(DEV))[0], *off(one * term.to(DEV), zero)[1:]]
    assert max(errors) <= 33, errors
