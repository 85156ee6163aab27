"""The token model's modules: plain forms on the CPU, the operators on the GPU, and a run
of them as they are used: prompts, single tokens, training steps, captured and not."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

import _model_ref as R
import ltc
import ltc_cuda

DEV = "cuda"
gpu = pytest.mark.gpu


class Model(nn.Module):
    """Tokens in, two mixing layers, scores out."""

    def __init__(self, vocab=61, dim=24, dtype=None):
        super().__init__()
        self.embed = ltc.TokenEmbedding(vocab, dim, scale=dim ** 0.5, dtype=dtype)
        self.layers = nn.ModuleList(ltc.SelectiveTimeConstant(dim, hidden=40, states=8, dtype=dtype)
                                    for _ in range(2))
        self.readout = ltc.TokenReadout(dim, vocab, dtype=dtype)

    def hidden(self, ids, states=None, cu=None):
        h, new = self.embed(ids), []
        for i, layer in enumerate(self.layers):
            o, s = layer(h, None if states is None else states[i], cu)
            h = h + o
            new.append(s)
        return h, new

    def forward(self, ids, targets):
        h, _ = self.hidden(ids)
        return self.readout.log_probs(h, targets)[0]

    def step(self, ids, states, slots=None):
        h = self.embed(ids)
        for layer, s in zip(self.layers, states):
            h = h + layer.step(h, s, slots)
        return h


def _model(device="cpu", dtype=None, seed=0):
    torch.manual_seed(seed)
    return Model(dtype=dtype).to(device)


def _ids(*shape, seed=1, V=61):
    return torch.randint(0, V, shape, generator=torch.Generator().manual_seed(seed))


def test_plain_layer_is_the_definition():
    torch.manual_seed(3)
    m = ltc.SelectiveTimeConstant(12, hidden=20, states=5, taps=3).double()
    x = torch.randn(2, 9, 12).double()
    out, (tail, h) = m(x)
    both = m.in_proj(x)
    u, t = R.conv(both[..., :20], m.conv_weight, m.conv_bias, act="silu")
    delta, B, C = m._selected(u)
    y, s = R.scan(u, delta, -torch.exp(m.A_log), B[:, :, None], C[:, :, None], m.D, both[..., 20:], m.dt_bias,
                  softplus=True)
    # the plain scan runs in float32: 9 tokens of some tens of roundings each
    assert torch.allclose(out, m.out_proj(y), atol=1e-5) and torch.allclose(tail, t)
    assert torch.allclose(h.double(), s, atol=1e-5)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_prompt_then_tokens_is_the_whole(device):
    """Tokens one by one after a prompt, in rows of a pool, against the whole sequence: off by
    the roundings of two orders of the same sums, some hundreds of 2^-24 at sizes of some
    tens, in float32."""
    m = _model(device).eval()
    ids = _ids(3, 30).to(device)
    with torch.no_grad():
        whole, _ = m.hidden(ids)
        start, states = m.hidden(ids[:, :17])
        slots = torch.tensor([4, 0, 2, -1], dtype=torch.int32, device=device)
        pools = [s.new_state(6) for s in m.layers]
        for (a, b), (pa, pb) in zip(states, pools):
            pa[slots[:3].long()], pb[slots[:3].long()] = a, b
        for t in range(17, 30):
            now = torch.cat([ids[:, t], torch.tensor([-1], device=device)])
            h = m.step(now, pools, slots)
            assert float((h[:3] - whole[:, t]).abs().max()) <= 2e-4
            assert float(h[3].abs().max()) == 0
        for _, b in pools:
            assert float(b[1].abs().max()) == 0 and float(b[5].abs().max()) == 0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_packed_is_each_sequence(device):
    m = _model(device).eval()
    ids = _ids(40).to(device)
    cu = torch.tensor([0, 11, 11, 12, 37], dtype=torch.int32, device=device)
    with torch.no_grad():
        h, states = m.hidden(ids, cu=cu)
        for s, (a, b) in enumerate(((0, 11), (11, 12), (12, 37))):
            one, st = m.hidden(ids[None, a:b])
            assert float((h[a:b] - one[0]).abs().max()) <= 2e-4
            k = (0, 2, 3)[s]
            for x, y in zip(states, st):
                assert float((x[1][k] - y[1][0]).abs().max()) <= 2e-4


def test_adjusted_on_the_cpu():
    torch.manual_seed(2)
    m = ltc.TokenReadout(6, 70)
    h = torch.randn(3, 6)
    ctx, prompt = torch.randint(-2, 72, (3, 20)), torch.tensor([0, 5, 20], dtype=torch.int32)
    ids, b = torch.randint(-1, 71, (3, 4)), torch.randn(3, 4)
    mask = torch.randint(-(1 << 31), 1 << 31, (3, 3)).to(torch.int32)
    got = m.adjusted(h, ctx, prompt, 1.3, 0.2, 0.4, ids, b, mask).double()
    want = R.adjust(m(h).detach(), ctx, prompt, 1.3, 0.2, 0.4, ids, b, mask)
    assert torch.equal(got.isinf(), want.isinf())
    assert float((got - want)[want.isfinite()].abs().max()) <= 20 * 2.0 ** -24 * 40


def test_absent_tokens_on_the_cpu():
    m = ltc.TokenEmbedding(5, 4, scale=2.0)
    out = m(torch.tensor([[1, -1], [-7, 4]]))
    out.sum().backward()
    assert torch.equal(out[0, 0], m.weight[1] * 2) and float(out[0, 1].abs().sum()) == 0
    assert torch.equal(m.weight.grad.sum(1), torch.tensor([0.0, 8.0, 0.0, 0.0, 8.0]))


@gpu
def test_gpu_is_the_cpu():
    """Outputs and every parameter's gradient; float32, whose roundings over 25 tokens, two
    layers and sums of a hundred terms stay under 1e-4 of the largest entry."""
    a, b = _model(), _model(DEV)
    ids, tgt = _ids(4, 25), _ids(4, 25, seed=2)
    ids[1, 20:] = -1
    tgt[1, 20:] = -1
    la, lb = a(ids, tgt), b(ids.to(DEV), tgt.to(DEV))
    assert float((la - lb.cpu()).abs().max()) <= 1e-4 * float(la.detach().abs().max())
    la.sum().backward()
    lb.sum().backward()
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        size = float(p.grad.abs().max())
        assert size > 0 and float((p.grad - q.grad.cpu()).abs().max()) <= 1e-4 * size, n


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_step(dtype):
    """Replays against eager steps on new data, bit for bit."""
    m = _model(DEV, dtype)
    ids, tgt = _ids(4, 32).to(DEV), _ids(4, 32, seed=2).to(DEV)

    class Wrapped(nn.Module):
        def __init__(self):
            super().__init__()
            self.m = m

        def forward(self, i, t):
            return self.m(i, t)

    weight = torch.randn(4, 32, device=DEV)
    step = ltc_cuda.CapturedStep(Wrapped(), (ids, tgt), lambda lp: lp * weight)
    for k in range(3):
        new = _ids(4, 32, seed=10 + k).to(DEV)
        step.inputs[0].copy_(new)
        step.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in step.grads]
        out = step.outputs.clone()
        params = [p for p in m.parameters()]
        lp = m(new, tgt)
        want = torch.autograd.grad(lp * weight, params, torch.ones_like(lp))
        assert torch.equal(out, lp.detach())
        for (n, _), a, b in zip(m.named_parameters(), got, want):
            assert torch.equal(a, b), n


@gpu
def test_decoding_under_a_mask():
    """Greedy decoding with penalties and a mask: what is chosen is allowed and best by the
    definition of the adjusted scores."""
    m = _model(DEV).eval()
    ids = _ids(2, 8).to(DEV)
    with torch.no_grad():
        h, states = m.hidden(ids)
        last, seen = h[:, -1], ids
        for t in range(6):
            allow = torch.randint(-(1 << 31), 1 << 31, (2, 2), generator=torch.Generator().manual_seed(t)).to(torch.int32)
            scores = m.readout.adjusted(last, seen, torch.full((2,), 8, dtype=torch.int32, device=DEV), 1.2, 0.1, 0.3,
                                        mask=allow.to(DEV))
            want = R.adjust(m.readout(last).cpu(), seen.cpu(), torch.tensor([8, 8]), 1.2, 0.1, 0.3, mask=allow)
            fin = want.isfinite()
            assert torch.equal(scores.cpu().isfinite(), fin)
            assert float((scores.cpu().double() - want)[fin].abs().max()) <= 1e-5
            lp, _, _, top = m.readout.log_probs(last, torch.zeros(2, dtype=torch.int64, device=DEV), top=1)
            nxt = scores.argmax(-1)
            for r in range(2):
                assert int(allow[r, int(nxt[r]) // 32]) >> (int(nxt[r]) % 32) & 1
            seen = torch.cat([seen, nxt[:, None]], 1)
            last = m.step(nxt, states)


@gpu
def test_a_module_of_another_type():
    """Turned to bfloat16 as a whole it runs, its scan's rates in float32 all the same."""
    m = _model(DEV).to(torch.bfloat16)
    h, states = m.hidden(_ids(2, 9).to(DEV))
    assert h.dtype == torch.bfloat16 and states[0][1].dtype == torch.float32
    h.float().sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for n, p in m.named_parameters()
               if "readout" not in n)
    m.step(_ids(2).to(DEV), [s.new_state(2) for s in m.layers])
