"""Log probabilities of given tokens and distillation from a teacher's top logits on the
GPU against float64: vocabulary sizes around the kernels' vectors and splits, types,
layouts, masked vocabularies, missing tokens and entries, ties, extremes, graphs."""

from __future__ import annotations

import pytest
import torch

import ltc_cuda
from _gpu_common import DEV, _native  # noqa: F401
import _seq_ref as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")
SIZES = [(1, 1), (1, 2), (3, 7), (5, 63), (2, 64), (4, 257), (3, 1000), (2, 8191), (2, 8192), (1, 50021),
         (1100, 130), (9, 131072)]


def _rows(N, V, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed + 31 * V + N)
    x = (torch.randn(N, V, generator=g) * scale).to(dtype)
    ids = torch.randint(0, V, (N,), generator=g)
    return x, ids, torch.randn(N, generator=g), torch.randn(N, generator=g) * 0.3, g


def _check_logprobs(x, ids, gp, ge, temperature=1.0, top=0, xd=None):
    val, tol = R.logprobs(x, ids, temperature, top, gp, ge)
    leaf = (x.to(DEV) if xd is None else xd).requires_grad_(True)
    res = ltc_cuda.ltc_token_logprobs(leaf, ids.to(DEV), top=top, temperature=temperature)
    grad, = torch.autograd.grad(res[:2], [leaf], [gp.to(DEV), ge.to(DEV)])
    names = ["logp", "ent"] + (["top_logp", "top_ids"] if top else []) + ["gx"]
    for name, got in zip(names, [t.detach() for t in res] + [grad]):
        R.close(got.cpu(), val[name], tol.get(name, 0.0), name)


@pytest.mark.parametrize("N,V", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_logprobs_sizes(N, V, dtype):
    x, ids, gp, ge, _ = _rows(N, V, dtype)
    _check_logprobs(x, ids, gp, ge, top=min(V, 5))


@pytest.mark.parametrize("top", [1, 2, 20, 31, 32])
@pytest.mark.parametrize("N,V", [(3, 40), (2, 600), (1, 40000), (1100, 600)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_with_ties(N, V, top, dtype):
    x, ids, gp, ge, g = _rows(N, V, dtype)
    x = torch.round(x)  # many equal logits, and -0 beside +0
    x[0, ::3] = -0.0
    _check_logprobs(x, ids, gp, ge, top=top)


@pytest.mark.parametrize("order", ["ascending", "descending", "equal", "spike"])
def test_top_orders(order):
    V = 5000
    x = {"ascending": torch.arange(V), "descending": -torch.arange(V), "equal": torch.zeros(V),
         "spike": torch.zeros(V)}[order].float().expand(2, V).contiguous() / 100
    if order == "spike":
        x[:, 4321] = 9.0
    _check_logprobs(x, torch.tensor([0, V - 1]), torch.randn(2), torch.randn(2), top=32)


@pytest.mark.parametrize("temperature", [0.25, 0.7, 1.0, 3.0])
def test_temperature(temperature):
    x, ids, gp, ge, _ = _rows(4, 3001, F32)
    _check_logprobs(x, ids, gp, ge, temperature, top=3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_masked_vocabularies(dtype):
    """-inf and the type's lowest value as masks; all but one token masked; fewer allowed
    tokens than alternatives."""
    x, ids, gp, ge, g = _rows(6, 700, dtype)
    low = torch.finfo(dtype).min
    x[0, 100:] = -INF
    x[1, :650] = low
    x[2] = -INF
    x[2, 5] = 1.0
    x[3] = low
    x[4, 3:] = -INF
    x[5, ::2] = low
    ids = torch.tensor([3, 660, 5, 0, 1, 1])
    _check_logprobs(x, ids, gp, ge, top=8)
    # a masked token was given: -inf, and its gradient is finite but for the entropy's none
    ids = torch.tensor([200, 1, 6, 699, 400, 0])
    _check_logprobs(x, ids, gp, torch.zeros_like(ge))


def test_large_logits_lose_nothing():
    x, ids, gp, ge, _ = _rows(4, 999, F32)
    _check_logprobs(x + 4096.0, ids, gp, ge)
    _check_logprobs(x * 1000, ids, gp, ge)


def test_rows_without_a_token_and_bad_ids():
    x, ids, gp, ge, _ = _rows(6, 130, F32)
    ids = torch.tensor([-100, 3, -1, 130, 2 ** 40, 129])
    x[0] = float("nan")  # never looked at for the gradient of a row without a token
    val, tol = R.logprobs(x, ids, 1.0, 0, gp, ge)
    leaf = x.to(DEV).requires_grad_(True)
    for i in (ids, ids.clamp(max=2 ** 31 - 1).int()):
        lp, en = ltc_cuda.ltc_token_logprobs(leaf, i.to(DEV))
        g, = torch.autograd.grad([lp, en], [leaf], [gp.to(DEV), ge.to(DEV)])
        assert lp[0] == 0 and en[0] == 0 and lp[2] == 0 and en[2] == 0
        assert torch.isnan(lp[3:5]).all() and torch.isnan(en[3:5]).all()
        assert (g[0] == 0).all() and (g[2] == 0).all() and torch.isnan(g[3:5]).all()
        for k in (1, 5):
            R.close(lp[k].cpu(), val["logp"][k], tol["logp"][k], "logp")
            R.close(g[k].cpu(), val["gx"][k], tol["gx"][k], "gx")


def test_rows_that_have_no_distribution_give_nan():
    x = torch.randn(5, 300, device=DEV)
    x[0, 7] = float("nan")
    x[1, 8] = INF
    x[2] = -INF
    lp, en, tl, ti = ltc_cuda.ltc_token_logprobs(x, torch.zeros(5, dtype=torch.long, device=DEV), top=4)
    assert torch.isnan(lp[:3]).all() and torch.isnan(en[:3]).all() and torch.isnan(tl[:3]).all()
    assert torch.isfinite(lp[3:]).all() and torch.isfinite(en[3:]).all() and torch.isfinite(tl[3:]).all()
    assert ((ti >= 0) & (ti < 300)).all()


def test_shapes_and_layouts():
    g = torch.Generator().manual_seed(5)
    full = torch.randn(2, 3, 2, 501, generator=g)
    ids = torch.randint(0, 400, (2, 3), generator=g)
    for view in (lambda t: t[:, :, 0, :400], lambda t: t[:, :, 1, 1:401], lambda t: t[:, :, 0, ::1][..., 100:500],
                 lambda t: t[:, :, 0, 1:].reshape(2, 3, 500)[..., ::1][..., :400],
                 lambda t: t.permute(0, 1, 3, 2)[..., 0][..., :400], lambda t: t[:, :, 0, 0:800:2][..., :250]):
        x = view(full.to(DEV))
        V = x.shape[-1]
        i = (ids % V).to(DEV)
        a = ltc_cuda.ltc_token_logprobs(x, i, top=3)
        val, tol = R.logprobs(x.cpu().reshape(6, V), i.cpu().reshape(6), 1.0, 3)
        assert a[0].shape == (2, 3) and a[2].shape == (2, 3, 3) and a[3].dtype == torch.int64
        for name, t in zip(("logp", "ent", "top_logp", "top_ids"), a):
            v = val[name].reshape(t.shape)
            R.close(t.cpu(), v, tol[name].reshape(t.shape) if name in tol else 0.0, name)
    # one row of all tokens, and no rows
    one = ltc_cuda.ltc_token_logprobs(full[0, 0, 0].to(DEV), torch.tensor(3, device=DEV))
    assert one[0].shape == ()
    none = torch.zeros(0, 9, device=DEV, requires_grad=True)
    res = ltc_cuda.ltc_token_logprobs(none, torch.zeros(0, dtype=torch.long, device=DEV), top=2)
    assert [t.shape[0] for t in res] == [0] * 4
    assert torch.autograd.grad(res[0].sum(), [none])[0].shape == (0, 9)


def _teacher(N, V, K, g, dtype, absent=0.0):
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    t = (torch.randn(N, K, generator=g) * 2 + 2).to(dtype)
    if absent:
        ids[torch.rand(N, K, generator=g) < absent] = -1
    return t, ids


def _check_distill(x, t, ids, gl, temperature=1.0):
    val, tol = R.distill(x, t, ids, temperature, gl)
    leaf = x.to(DEV).requires_grad_(True)
    for i in (ids, ids.int()):
        loss = ltc_cuda.ltc_top_distill(leaf, t.to(DEV), i.to(DEV), temperature=temperature)
        grad, = torch.autograd.grad(loss, [leaf], [gl.to(DEV)])
        R.close(loss.detach().cpu(), val["loss"], tol["loss"], "loss")
        R.close(grad.cpu(), val["gx"], tol["gx"], "gx")


@pytest.mark.parametrize("N,V", SIZES)
@pytest.mark.parametrize("dtype,tdtype", [(F32, F32), (BF16, F32), (F16, BF16)])
def test_distill_sizes(N, V, dtype, tdtype):
    x, _, gl, _, g = _rows(N, V, dtype)
    t, ids = _teacher(N, V, min(V, 7), g, tdtype)
    _check_distill(x, t, ids, gl)


@pytest.mark.parametrize("K", [1, 2, 64, 255, 256, 257, 1024])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_distill_entries(K, temperature):
    x, _, gl, _, g = _rows(3, 2000, F32)
    t, ids = _teacher(3, 2000, K, g, F32, absent=0.3)
    _check_distill(x, t, ids, gl, temperature)


def test_distill_repeated_absent_and_masked_entries():
    x, _, gl, _, g = _rows(7, 300, F32)
    t, ids = _teacher(7, 300, 6, g, F32)
    ids[0] = 17                      # one id in every place
    ids[1] = -1                      # a row without entries
    ids[2, 1:] = -5
    t[3] = -INF                      # entries of no weight
    t[4, :3] = -INF
    t[5] = torch.finfo(F32).min      # equal ones
    x[6, :200] = -INF                # a masked vocabulary that holds the entries
    ids[6] = torch.arange(200, 206)
    _check_distill(x, t, ids, gl)
    # the student gives an entry no probability: the loss is infinite
    x[6, 203] = -INF
    _check_distill(x, t, ids, gl)
    ids[2, 0] = 300                  # an id past the vocabulary
    val, _ = R.distill(x, t, ids, 1.0)
    loss = ltc_cuda.ltc_top_distill(x.to(DEV), t.to(DEV), ids.to(DEV))
    assert torch.isnan(loss[2]) and torch.equal(torch.isnan(loss.cpu()), torch.isnan(val["loss"]))


def test_distill_teacher_that_is_not_a_number():
    x = torch.randn(3, 50, device=DEV, requires_grad=True)
    t = torch.randn(3, 4, device=DEV)
    ids = torch.arange(4, device=DEV).expand(3, 4)
    t[0, 1] = float("nan")
    t[1, 2] = INF
    loss = ltc_cuda.ltc_top_distill(x, t, ids)
    g, = torch.autograd.grad(loss.sum(), [x])
    assert torch.isnan(loss[:2]).all() and torch.isfinite(loss[2])
    assert torch.isnan(g[:2]).all() and torch.isfinite(g[2]).all()


def test_gradients_against_differences():
    """Central differences of the float64 references' own values."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 6, generator=g).double()
    ids, gp, ge = torch.tensor([1, 4]), torch.randn(2, generator=g).double(), torch.randn(2, generator=g).double()
    t, tid = torch.randn(2, 3, generator=g).double(), torch.tensor([[0, 2, 2], [5, -1, 3]])
    lv, _ = R.logprobs(x, ids, 0.8, 0, gp, ge)
    dv, _ = R.distill(x, t, tid, 1.7, gp)

    def lose(z):
        v, _ = R.logprobs(z, ids, 0.8)
        return float((v["logp"] * gp + v["ent"] * ge).sum())

    def teach(z):
        return float((R.distill(z, t, tid, 1.7)[0]["loss"] * gp).sum())

    for f, want in ((lose, lv["gx"]), (teach, dv["gx"])):
        for i in range(x.numel()):
            up, dn = x.clone(), x.clone()
            up.view(-1)[i] += 1e-5
            dn.view(-1)[i] -= 1e-5
            assert abs((f(up) - f(dn)) / 2e-5 - float(want.reshape(-1)[i])) < 1e-8


def test_same_results_every_time_and_in_graphs():
    x, ids, gp, ge, g = _rows(3, 40000, BF16)
    t, tid = _teacher(3, 40000, 40, g, F32, 0.2)
    leaf = x.to(DEV).requires_grad_(True)
    ids, gp, ge, t, tid = (v.to(DEV) for v in (ids, gp, ge, t, tid))

    def step():
        r = ltc_cuda.ltc_token_logprobs(leaf, ids, top=9)
        d = ltc_cuda.ltc_top_distill(leaf, t, tid, temperature=2.0)
        return [*r, d, *torch.autograd.grad(r[:2], [leaf], [gp, ge]), *torch.autograd.grad(d, [leaf], [gp])]

    eager = [v.detach().clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(again, eager):
        assert torch.equal(p.detach(), q)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    again = None  # no eager graph of the leaf may live during a capture
    with torch.cuda.graph(graph):
        a = step()
    with torch.cuda.graph(other):
        b = step()
    for i in range(4):
        if i == 2:
            with torch.no_grad():
                leaf.mul_(0.5)
            eager = [v.detach().clone() for v in step()]
        graph.replay()
        torch.randn(1000, device=DEV).sum().item()
        other.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(a, b, eager):
            assert torch.equal(p.detach(), r) and torch.equal(q.detach(), r)


def test_refusals():
    f, d = ltc_cuda.ltc_token_logprobs, ltc_cuda.ltc_top_distill
    x = torch.zeros(2, 9, device=DEV)
    i = torch.zeros(2, dtype=torch.long, device=DEV)
    t, ti = torch.zeros(2, 3, device=DEV), torch.zeros(2, 3, dtype=torch.long, device=DEV)
    for err, call in [
            (ValueError, lambda: f(x, i[:1])),
            (ValueError, lambda: f(x, i, top=10)),
            (ValueError, lambda: f(x, i, top=-1)),
            (ValueError, lambda: f(torch.zeros(2, 90, device=DEV), i, top=33)),
            (ValueError, lambda: f(x, i, temperature=0.0)),
            (ValueError, lambda: f(x, i, temperature=float("nan"))),
            (RuntimeError, lambda: f(x, i, temperature=float("inf"))),
            (ValueError, lambda: f(x.cpu(), i.cpu())),
            (ValueError, lambda: f(x, i.cpu())),
            (ValueError, lambda: f(x[:, :0], i)),
            (TypeError, lambda: f(x.double(), i)),
            (TypeError, lambda: f(x, i.float())),
            (ValueError, lambda: d(x, t[:, :2], ti)),
            (ValueError, lambda: d(x, t[:1], ti[:1])),
            (ValueError, lambda: d(x, t[:, :0], ti[:, :0])),
            (ValueError, lambda: d(x, t, ti, temperature=-1.0)),
            (ValueError, lambda: d(x, t.cpu(), ti)),
            (ValueError, lambda: d(x, torch.zeros(2, 1025, device=DEV),
                                   torch.zeros(2, 1025, dtype=torch.long, device=DEV))),
            (ValueError, lambda: d(x, t.clone().requires_grad_(True), ti)),
            (TypeError, lambda: d(x, t.long(), ti)),
            (TypeError, lambda: d(x, t, ti.short()))]:
        with pytest.raises(err):
            call()
