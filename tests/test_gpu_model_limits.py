"""The token model's operators on tensors of more than 2^31 elements: the first and the last
tokens, rows or ids against their definitions. Tolerances are those of each operator's own
file."""

from __future__ import annotations

import pytest
import torch

import _model_ref as R
import ltc_cuda
import test_gpu_adjust_logits as A
import test_gpu_causal_conv as C
import test_gpu_selective_scan as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF16 = torch.bfloat16
N, H = 1_050_000, 2056


def _rand(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


@pytest.mark.parametrize("packed", [False, True])
def test_conv(packed):
    g = torch.Generator(DEV).manual_seed(1)
    x, go = _rand(g, N, H).requires_grad_(True), _rand(g, N, H)
    w = _rand(g, H, 4).requires_grad_(True)
    cu = torch.tensor([0, N - 450, N], dtype=torch.int32, device=DEV) if packed else None
    out, hf = ltc_cuda.ltc_causal_conv(x if packed else x[None], w, cu_seqlens=cu)
    out = out.view(N, H)
    gx, = torch.autograd.grad(out, [x], go)
    assert torch.equal(hf[-1], x[-3:].detach())
    n = 60
    for part, rows in ((slice(N - n, N), slice(n - 40, n)), (slice(0, n), slice(0, 40))):
        xs = x[part].detach().cpu().double()[None].requires_grad_(True)
        want, _ = R.conv(xs, w.detach().cpu().double())
        ref, = torch.autograd.grad(want, [xs], go[part].cpu().double()[None])
        ab = xs.detach().abs().requires_grad_(True)
        mag, _ = R.conv(ab, w.detach().cpu().double().abs())
        gmag, = torch.autograd.grad(mag, [ab], go[part].cpu().double().abs()[None])
        C._close(out[part][rows], want[0, rows], mag.detach()[0, rows], "bf16", 4 + 16)
        C._close(gx[part][rows], ref[0, rows], gmag[0, rows], "bf16", 4 + 24 + 4)


def test_scan():
    """Decays of at most exp(-step) a token, steps of 0.8 on average: what lies 300 tokens
    off adds nothing that float32 holds."""
    g = torch.Generator(DEV).manual_seed(2)
    K = 4
    t = {"x": _rand(g, 1, N, H), "delta": _rand(g, 1, N, H), "B": _rand(g, 1, N, K), "C": _rand(g, 1, N, K)}
    t["A"] = -1 - 3 * torch.rand(H, K, generator=g, device=DEV)
    go = _rand(g, 1, N, H)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    out, hf = ltc_cuda.ltc_selective_scan(**leaves, delta_softplus=True)
    names = ("x", "delta", "B", "C")
    grads = dict(zip(names, torch.autograd.grad(out, [leaves[k] for k in names], go)))
    n, keep = 400, 60
    for part, rows in ((slice(N - n, N), slice(n - keep, n)), (slice(0, n), slice(0, keep))):
        one = {k: (v.detach() if k == "A" else v.detach()[:, part]).cpu() for k, v in t.items()}
        one["B"], one["C"] = one["B"][:, :, None], one["C"][:, :, None]
        one.update(D=None, z=None, bias=None, state=None)
        d = {k: None if v is None else v.double().requires_grad_(True) for k, v in one.items()}
        want, whf = R.scan(d["x"], d["delta"], d["A"], d["B"], d["C"], softplus=True)
        gp = go[:, part].cpu()
        ref = torch.autograd.grad(want, [d[k] for k in names], gp.double())
        mo, mh, mg = S._sizes(one, None, True, gp, torch.zeros(1, H, K))
        count = 40 * n + 16 + K
        S._close(out[0, part][rows], want[0, rows], mo[0, rows], "bf16", count, "out")
        for k, r in zip(names, ref):
            got = grads[k][0, part][rows]
            S._close(got, r.view(1, n, -1)[0, rows], mg[k].view(1, n, -1)[0, rows], "bf16",
                     2 * count + 32 + H, k)
        if part.start > 0:
            S._close(hf, whf, mh, "fp32", count, "state")


def test_steps():
    P = N
    g = torch.Generator(DEV).manual_seed(3)
    slots = torch.tensor([0, P - 1, P - 2, -1], dtype=torch.int32, device=DEV)
    x, w = _rand(g, 4, H, dtype=torch.float32), _rand(g, H, 2, dtype=torch.float32)
    pool = torch.zeros(P, 1, H, device=DEV)
    pool[slots[:3].long(), 0] = _rand(g, 3, H, dtype=torch.float32)
    small = pool[slots[:3].long()].clone()
    out = ltc_cuda.ltc_causal_conv_step(x, w, pool, slots=slots)
    assert torch.equal(out[:3], ltc_cuda.ltc_causal_conv_step(x[:3], w, small))
    assert torch.equal(pool[slots[:3].long()], small) and not out[3].any() and not pool[1:P - 2].any()
    K = 4
    pool = torch.zeros(P, H // K, K, device=DEV)
    pool[slots[:3].long()] = _rand(g, 3, H // K, K, dtype=torch.float32)
    small = pool[slots[:3].long()].clone()
    one = {"x": x[:, :H // K], "delta": x[:, :H // K].abs(), "B": x[:, :K], "C": x[:, K:2 * K]}
    rates = -torch.rand(H // K, K, generator=g, device=DEV)
    out = ltc_cuda.ltc_selective_scan_step(**one, A=rates, state=pool, slots=slots)
    assert torch.equal(out[:3], ltc_cuda.ltc_selective_scan_step(**{k: v[:3] for k, v in one.items()}, A=rates,
                                                                 state=small))
    assert torch.equal(pool[slots[:3].long()], small) and not out[3].any() and not pool[1:P - 2].any()


def test_embed():
    g = torch.Generator(DEV).manual_seed(4)
    # many rows of the table
    table = _rand(g, N, H).requires_grad_(True)
    ids = torch.tensor([N - 1, 0, N - 1, N - 2, 5, -1, N], device=DEV)
    out = ltc_cuda.ltc_embed(table, ids)
    assert torch.equal(out[:5], table.detach()[ids[:5]]) and not out[5].any() and bool(out[6].isnan().all())
    go = _rand(g, 7, H)
    grad, = torch.autograd.grad(out, [table], go)
    both = go[0].double() + go[2].double()
    tol = (go[0].abs() + go[2].abs()).double() * 2 * U + R.half_step("bf16") * both.abs() * (1 + 2 * U)
    assert bool(((grad[N - 1].double() - both).abs() <= tol).all())
    assert torch.equal(grad[0], go[1]) and torch.equal(grad[N - 2], go[3]) and torch.equal(grad[5], go[4])
    assert not grad[1:5].any() and not grad[6:N - 2].any()
    del table, out, grad
    # many ids
    table = _rand(g, 50, H).requires_grad_(True)
    ids = torch.randint(0, 50, (N,), generator=g, device=DEV)
    out = ltc_cuda.ltc_embed(table, ids)
    for part in (slice(0, 3), slice(N - 3, N)):
        assert torch.equal(out[part], table.detach()[ids[part]])
    go = _rand(g, N, H)
    grad, = torch.autograd.grad(out, [table], go)
    for cols in (slice(0, 8), slice(H - 8, H)):
        d = go[:, cols].double()
        ref = torch.zeros(50, 8, dtype=torch.float64, device=DEV).index_add_(0, ids, d)
        mag = torch.zeros(50, 8, dtype=torch.float64, device=DEV).index_add_(0, ids, d.abs())
        err = (torch.bincount(ids, minlength=50).double()[:, None] + 1) * U * mag
        assert bool(((grad[:, cols].double() - ref).abs() <= err + R.half_step("bf16") * (ref.abs() + err)).all())


def test_adjust():
    rows, V = 17000, 128256
    g = torch.Generator(DEV).manual_seed(5)
    x = _rand(g, rows, V)
    ids = torch.randint(0, V, (rows, 40), generator=g, device=DEV)
    bid, b = torch.tensor([V - 1, 3], device=DEV), torch.tensor([1.5, -2.0], device=DEV)
    got = ltc_cuda.ltc_adjust_logits(x, ids, repetition=1.3, frequency=0.2, presence=0.5, bias_ids=bid, bias=b)
    for part in (slice(0, 2), slice(rows - 2, rows)):
        c = x[part].cpu()
        want = R.adjust(c, ids[part].cpu(), None, 1.3, 0.2, 0.5, bid.cpu().expand(2, 2), b.cpu().expand(2, 2))
        A._close(got[part], want, c.double().abs() * 2 + 80 + 1 + 3.5, "bf16", 2)
