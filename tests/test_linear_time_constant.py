"""LinearTimeConstant and TokenReadout: against TrueLiquidTimeConstant, of which the
first is the case without recurrent synapses, against plain torch, and used together."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import ltc
import ltc_cuda

GPU = pytest.param("cuda", marks=pytest.mark.gpu)


def _layers(D, H, seed=0, mapping="affine"):
    """The layer, and the same as a TrueLiquidTimeConstant of one unfold without
    recurrent synapses."""
    torch.manual_seed(seed)
    lin = ltc.LinearTimeConstant(D, H, input_mapping=mapping)
    full = ltc.TrueLiquidTimeConstant(D, H, ode_unfolds=1, input_mapping=mapping)
    with torch.no_grad():
        for p in lin.parameters():
            p.add_(0.05 * torch.randn_like(p))
        full.sparsity_mask.zero_()
        full.erev.zero_()
    missing, unexpected = full.load_state_dict(lin.state_dict(), strict=False)
    assert not unexpected and set(missing) == {"w", "mu", "sigma", "erev", "sparsity_mask"}
    return lin, full


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("mapping", ["affine", "linear", "none"])
@pytest.mark.parametrize("B,T,D,H", [(1, 1, 3, 4), (3, 9, 10, 17), (2, 200, 8, 64)])
def test_is_the_layer_without_recurrent_synapses(device, B, T, D, H, mapping):
    lin, full = _layers(D, H, mapping=mapping)
    lin, full = lin.to(device), full.to(device)
    x = torch.randn(B, T, D, device=device, requires_grad=True)
    h0 = (torch.randn(B, H, device=device) * 0.3).requires_grad_(True)
    go, gh = torch.randn(B, T, H, device=device), torch.randn(B, H, device=device)
    got = []
    for m in (lin, full):
        out, (h, c) = m(x, (h0, h0))
        assert h is c
        names = [n for n, _ in lin.named_parameters()]
        ps = dict(m.named_parameters())
        grads = torch.autograd.grad([out, h], [x, h0, *(ps[n] for n in names)], [go, gh])
        got.append([out, h, *grads])
    # two fp32 evaluations of one formula, by different routes (a division here, a
    # sigmoid of logarithms there): each within a few tens of roundings per step of
    # a sequence whose memory is a few steps
    for a, b in zip(*got):
        scale = float(b.detach().abs().max()) + 1e-6
        assert float((a - b).detach().abs().max()) <= 2e-4 * scale


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_packed_sequences_and_steps_follow_the_batch(device):
    lin = _layers(6, 20)[0].to(device)
    lengths = [5, 0, 12, 1]
    cu = torch.tensor([0, 5, 5, 17, 18], dtype=torch.int32, device=device)
    x = torch.randn(18, 6, device=device)
    h0 = torch.randn(4, 20, device=device)
    out, (h, _) = lin(x, (h0, h0), cu_seqlens=cu)
    pool = torch.zeros(9, 20, device=device)
    rows = [7, 2, 0, 4]
    pool[rows] = h0
    for s, n in enumerate(lengths):
        lo = int(cu[s])
        if n == 0:
            assert torch.equal(h[s], h0[s])
            continue
        o, (hs, _) = lin(x[None, lo:lo + n], (h0[s:s + 1], None))
        torch.testing.assert_close(out[lo:lo + n], o[0], rtol=1e-5, atol=1e-6)
        torch.testing.assert_close(h[s], hs[0], rtol=1e-5, atol=1e-6)
    # the same tokens one by one: streams that have ended are padding
    for t in range(max(lengths)):
        live = [t < n for n in lengths]
        xs = torch.stack([x[min(int(cu[s]) + t, 17)] for s in range(4)])
        slots = torch.tensor([r if on else -1 for r, on in zip(rows, live)], dtype=torch.int32,
                             device=device)
        o = lin.step(xs, pool, slots)
        for s in range(4):
            if live[s]:
                torch.testing.assert_close(o[s], out[int(cu[s]) + t], rtol=1e-5, atol=1e-6)
            else:
                assert not o[s].any()
    torch.testing.assert_close(pool[rows], h, rtol=1e-5, atol=1e-6)
    assert not pool[[1, 3, 5, 6, 8]].any()


class _Model(torch.nn.Module):
    """Tokens -> embedding -> layer -> readout."""

    def __init__(self, vocab, D, H, dtype=None):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, D)
        self.layer = ltc.LinearTimeConstant(D, H)
        self.readout = ltc.TokenReadout(H, vocab, dtype=dtype)

    def forward(self, x):
        return self.layer(x)[0]


def _plain_losses(logits, ids, t, tid, tau):
    lq = torch.log_softmax(logits.float() / tau, -1)
    p = torch.softmax(t.float() / tau, -1)
    kl = tau * tau * (p * (torch.log(p) - lq.gather(-1, tid))).sum(-1)
    l1 = torch.log_softmax(logits.float(), -1)
    ent = -(l1.exp() * l1).sum(-1)
    return kl, l1.gather(-1, ids.unsqueeze(-1)).squeeze(-1), ent


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_readout_against_plain_torch(device):
    torch.manual_seed(2)
    m = _Model(50, 8, 16).to(device)
    x = torch.randn(3, 7, 8, device=device)
    ids = torch.randint(0, 50, (3, 7), device=device)
    tid = torch.argsort(torch.rand(3, 7, 50, device=device), -1)[..., :5]
    t = torch.randn(3, 7, 5, device=device)
    ps = list(m.parameters())[1:]
    h = m(x)
    loss = m.readout.distill(h, t, tid, temperature=2.0)
    lp, ent, tl, ti = m.readout.log_probs(h, ids, top=4)
    got = torch.autograd.grad((loss - lp + 0.1 * ent).sum(), ps)
    logits = m.readout(m(x))
    kl, l1, e1 = _plain_losses(logits, ids, t, tid, 2.0)
    want = torch.autograd.grad((kl - l1 + 0.1 * e1).sum(), ps)
    for a, b in zip((loss, lp, ent), (kl, l1, e1)):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    assert torch.equal(ti, torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :4])
    torch.testing.assert_close(tl, torch.log_softmax(logits, -1).gather(-1, ti), rtol=1e-5, atol=1e-5)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,T,D,H", [
    (torch.float32, 4, 150, 16, 32), (torch.bfloat16, 4, 150, 16, 32),
    # many rows, and many inputs: what sums over either is replayed like the rest
    (torch.float32, 16, 2048, 64, 96), (torch.float32, 2, 120, 1023, 1100)])
def test_a_captured_distillation_step_and_serving(dtype, B, T, D, H):
    """Training as a program does it, one graph per step, then scoring and decoding."""
    torch.manual_seed(3)
    V, K = 700, 12
    m = _Model(V, D, H, dtype).cuda()
    x, x2 = (torch.randn(B, T, D, device="cuda") for _ in range(2))
    tid = torch.argsort(torch.rand(B, T, V, device="cuda"), -1)[..., :K].contiguous()
    tid[0, 3] = -1
    t = torch.randn(B, T, K, device="cuda")
    ids = torch.randint(0, V, (B, T), device="cuda")
    ids[1, 100:] = -100
    # a loss of each token: torch's mean over many is replayed wrongly in a graph
    share = torch.full((B, T), 1.0 / (B * T), device="cuda")

    def loss_fn(h):
        lp, ent = m.readout.log_probs(h, ids)
        return share * (m.readout.distill(h, t, tid, temperature=2.0) - 0.1 * (lp + ent))

    def eager(xx):
        loss = loss_fn(m(xx))
        ps = [p for p in m.parameters()]
        g = torch.autograd.grad(loss, ps, torch.ones_like(loss), allow_unused=True)
        return [loss.detach().clone()] + [v.clone() for v in g if v is not None]

    want, want2 = eager(x), eager(x2)
    for v in want:
        assert torch.isfinite(v).all() and v.any()
    step = ltc_cuda.CapturedStep(m, (x.clone(),), loss_fn)
    for r in range(4):
        src, w = (x, want) if r % 2 == 0 else (x2, want2)
        step.inputs[0].copy_(src)
        loss = step.replay()
        torch.cuda.synchronize()
        used = [p.grad for n, p in m.named_parameters() if n != "embed.weight"]
        for a, b in zip([loss, *used], w):
            assert torch.equal(a, b)
        torch.randn(1000, device="cuda").sum().item()
    # scoring, then the same tokens one by one from the carried states
    with torch.no_grad():
        out = m(x)
        lp, ent, tl, ti = m.readout.log_probs(out, ids, top=3)
        state = torch.zeros(B, H, device="cuda")
        for s in range(min(T, 150)):
            o = m.layer.step(x[:, s], state)
            a = m.readout.log_probs(o, ids[:, s], top=3)
            # half steps of the logits' type, where the states differ in their last bits
            tol = 0.05 if dtype == torch.bfloat16 else 1e-4
            torch.testing.assert_close(a[0], lp[:, s], rtol=tol, atol=tol)
            torch.testing.assert_close(a[2], tl[:, s], rtol=tol, atol=tol)
    assert not lp[1, 100:].any() and not ent[1, 100:].any()
