"""The embedding and the gradient of its table against sums in 64 bits: every path of the
sort (one tile, several, many), runs inside and across pieces, absent and foreign ids.

Tolerances: an output is one product, rounded to float32 and to its type. A gradient adds
its k tokens one after the other or piece by piece, k roundings of half a step of 2^-24 of
the sum of sizes at most, one more for the scale, and half a step of its type."""

from __future__ import annotations

import pytest
import torch

import _model_ref as R
import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _check(ids, V, H, dtype, scale, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = R.TYPES[dtype]
    table = torch.randn(V, H, generator=g, device=DEV).to(dt).requires_grad_(True)
    out = ltc_cuda.ltc_embed(table, ids, scale)
    assert out.shape == (*ids.shape, H) and out.dtype == dt
    flat = ids.reshape(-1).long()
    there = (flat >= 0) & (flat < V)
    got, o = out.detach().reshape(-1, H).double(), table.detach().double()
    want = o[flat[there]] * torch.tensor(scale).double().item()
    tol = want.abs() * (R.half_step(dtype) + 2 * U) + torch.finfo(dt).tiny
    assert bool(((got[there] - want).abs() <= tol).all())
    assert float(got[flat < 0].abs().sum()) == 0 and bool(got[flat >= V].isnan().all())
    go = torch.randn(out.shape, generator=g, device=DEV).to(dt)
    grad, = torch.autograd.grad(out, [table], go)
    again, = torch.autograd.grad(ltc_cuda.ltc_embed(table, ids, scale), [table], go)
    assert torch.equal(grad, again)
    d = go.reshape(-1, H).double()[there]
    ref = torch.zeros(V, H, dtype=torch.float64, device=DEV).index_add_(0, flat[there], d) * scale
    mag = torch.zeros(V, H, dtype=torch.float64, device=DEV).index_add_(0, flat[there], d.abs()) * abs(scale)
    k = torch.bincount(flat[there], minlength=V).double()[:, None]
    err = (k + 1) * U * mag
    tol = err + R.half_step(dtype) * (ref.abs() + err) + torch.finfo(dt).tiny
    off = (grad.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert float(grad[k[:, 0] == 0].abs().sum()) == 0
    return grad


def _ids(n, V, seed=1, text=True):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    ids = (torch.exp(u * torch.log(torch.tensor(V + 1.0, dtype=torch.float64))) - 1).long() if text else (u * V).long()
    return ids.clamp(0, V - 1).to(DEV)


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 1000, 4095, 4096, 4097, 9000])
@pytest.mark.parametrize("V,H,dtype", [(1, 4, "fp32"), (7, 33, "bf16"), (1000, 8, "fp16"), (1500, 1, "fp32")])
def test_sizes(n, V, H, dtype):
    _check(_ids(n, V), V, H, dtype, 1.0)


@pytest.mark.parametrize("V,H", [(1023, 40), (1024, 40), (1025, 40), (70000, 16), (1 << 20, 4), (1100000, 2)])
def test_vocabularies(V, H):
    """One digit, two and three."""
    ids = torch.cat([_ids(6000, V, text=False), torch.tensor([0, V - 1, V - 1], device=DEV)])
    _check(ids, V, H, "fp32", 2.5)


def test_many_tiles():
    """More tiles than a workgroup adds up itself."""
    assert 300000 > 64 * 4096
    _check(_ids(300000, 5000), 5000, 8, "bf16", 0.125)


@pytest.mark.parametrize("H,dtype", [(300, "bf16"), (2048, "bf16"), (2500, "fp32"), (4100, "fp16")])
def test_widths(H, dtype):
    _check(_ids(500, 90), 90, H, dtype, H ** 0.5)


@pytest.mark.parametrize("n", [64, 128, 200, 5000])
def test_one_id(n):
    """A run over all pieces, and one that ends in one."""
    ids = torch.full((n,), 3, device=DEV)
    _check(ids, 5, 12, "fp32", 1.0)
    ids[n // 2 + 1:] = 4
    ids[:3] = 0
    _check(ids, 5, 12, "fp32", -1.5)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_absent_and_foreign(kind):
    ids = _ids(700, 50).to(kind)
    ids[::7], ids[3::11], ids[5::13] = -1, 50, -(1 << 31)
    if kind == torch.int64:
        ids[9::17], ids[10::19] = 1 << 40, -(1 << 62)
        ids[12::23] = (1 << 32) + 4
    _check(ids.view(7, 100), 50, 24, "bf16", 1.0)
    _check(torch.full((9,), -1, dtype=kind, device=DEV), 50, 24, "fp32", 1.0)
    _check(torch.full((9,), 50, dtype=kind, device=DEV), 50, 24, "fp32", 1.0)


def test_layouts_and_streams():
    g = torch.Generator().manual_seed(2)
    big = torch.randn(60, 40, generator=g).to(DEV)
    ids = _ids(300, 60).view(10, 30)
    a = ltc_cuda.ltc_embed(big[:, 4:28], ids.t())
    assert torch.equal(a, ltc_cuda.ltc_embed(big[:, 4:28].contiguous(), ids.t().contiguous()))
    assert torch.equal(ltc_cuda.ltc_embed(big.t(), ids % 40), ltc_cuda.ltc_embed(big.t().contiguous(), ids % 40))
    assert ltc_cuda.ltc_embed(big, torch.tensor(5, device=DEV)).shape == (40,)
    leaf = big.clone().requires_grad_(True)

    def run(go):
        o = ltc_cuda.ltc_embed(leaf[:, 4:28], ids)
        return torch.autograd.grad(o, [leaf], go)[0]

    wide = torch.randn(10, 30, 48, generator=g).to(DEV)
    want = run(wide[..., :24].contiguous())
    assert torch.equal(run(wide[..., :24]), want)
    tr = wide[..., :24].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(run(tr), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(wide[..., :24])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    o = ltc_cuda.ltc_embed(leaf, ids)
    s, = torch.autograd.grad(o.sum(), [leaf])
    assert torch.equal(s, torch.bincount(ids.view(-1), minlength=60).float()[:, None].expand(60, 40))


def test_non_finite_gradients_stay_in_their_rows():
    ids = _ids(500, 30)
    table = torch.randn(30, 16, device=DEV, requires_grad=True)
    go = torch.randn(500, 16, device=DEV)
    clean, = torch.autograd.grad(ltc_cuda.ltc_embed(table, ids), [table], go)
    go[17] = float("nan")
    go[18, 3] = float("inf")
    bad, = torch.autograd.grad(ltc_cuda.ltc_embed(table, ids), [table], go)
    rows = torch.ones(30, dtype=torch.bool, device=DEV)
    rows[ids[17]] = rows[ids[18]] = False
    assert torch.equal(bad[rows], clean[rows]) and bool(bad[ids[17]].isnan().all())


def test_refusals():
    t, ids = torch.randn(5, 4, device=DEV), torch.tensor([1, 2], device=DEV)
    for bad, exc in ((lambda: ltc_cuda.ltc_embed(t.cpu(), ids.cpu()), ValueError),
                     (lambda: ltc_cuda.ltc_embed(t, ids.cpu()), ValueError),
                     (lambda: ltc_cuda.ltc_embed(t.double(), ids), TypeError),
                     (lambda: ltc_cuda.ltc_embed(t, ids.float()), TypeError),
                     (lambda: ltc_cuda.ltc_embed(t[0], ids), ValueError),
                     (lambda: ltc_cuda.ltc_embed(t[:0], ids), ValueError),
                     (lambda: ltc_cuda.ltc_embed(t, ids, float("inf")), ValueError),
                     (lambda: ltc_cuda.ltc_embed(t, ids, 1e39), ValueError)):
        with pytest.raises(exc):
            bad()
    leaf = t.requires_grad_(True)
    out = ltc_cuda.ltc_embed(leaf, ids)
    g, = torch.autograd.grad(out.sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()
