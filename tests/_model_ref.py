"""Definitions of the token model's operators in 64 bits, token by token, for the tests."""

from __future__ import annotations

import math

import torch

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(t) -> float:
    """Largest relative error of one rounding to a type."""
    return torch.finfo(TYPES[t] if isinstance(t, str) else t).eps / 2


def runs_of(x, cu):
    """(rows' index in a (sequences, ...) tensor, tokens of x) of every sequence."""
    if cu is None:
        return [(b, lambda v, b=b: v[b]) for b in range(x.shape[0])]
    c = cu.tolist()
    return [(s, lambda v, s=s: v[c[s]:c[s + 1]]) for s in range(len(c) - 1)]


def silu(v):
    return v / (1.0 + torch.exp(-v))


def conv(x, w, bias=None, state=None, cu=None, act=None):
    """Differentiable; out in x's shape and the final state."""
    K = w.shape[1]
    n = x.shape[0] if cu is None else cu.numel() - 1
    outs, tails = [], []
    for s, of in runs_of(x, cu):
        seq = of(x)
        before = x.new_zeros(K - 1, x.shape[-1]) if state is None else state[s]
        line = torch.cat([before, seq])
        y = x.new_zeros(seq.shape)
        for t in range(seq.shape[0]):
            v = (line[t:t + K] * w.t()).sum(0)
            v = v if bias is None else v + bias
            y = torch.cat([y[:t], (silu(v) if act else v)[None], y[t + 1:]])
        outs.append(y)
        tails.append(line[seq.shape[0]:])
    hf = torch.stack(tails) if n else x.new_zeros(0, K - 1, x.shape[-1])
    if cu is None:
        return (torch.stack(outs) if n else torch.zeros_like(x)), hf
    lead, end = int(cu[0]), int(cu[-1])
    return torch.cat([x.new_zeros(lead, x.shape[-1]), *outs,
                      x.new_zeros(x.shape[0] - end, x.shape[-1])]), hf


def scan(x, delta, A, B, C, D=None, z=None, bias=None, state=None, cu=None, softplus=False):
    """Differentiable; B and C (..., G, N)."""
    H, N = A.shape
    G = B.shape[-2]
    n = x.shape[0] if cu is None else cu.numel() - 1

    def wide(v):
        return v.repeat_interleave(H // G, 0)

    outs, finals = [], []
    for s, of in runs_of(x, cu):
        h = x.new_zeros(H, N) if state is None else state[s]
        xs, ds, bs, cs = of(x), of(delta), of(B), of(C)
        ys = []
        for t in range(xs.shape[0]):
            dt = ds[t] if bias is None else ds[t] + bias
            if softplus:
                dt = torch.logaddexp(dt, torch.zeros_like(dt))
            h = torch.exp(dt[:, None] * A) * h + (dt * xs[t])[:, None] * wide(bs[t])
            y = (h * wide(cs[t])).sum(-1)
            if D is not None:
                y = y + D * xs[t]
            if z is not None:
                y = y * silu(of(z)[t])
            ys.append(y)
        outs.append(torch.stack(ys) if ys else x.new_zeros(0, H))
        finals.append(h)
    hf = torch.stack(finals) if n else x.new_zeros(0, H, N)
    if cu is None:
        return (torch.stack(outs) if n else torch.zeros_like(x)), hf
    lead, end = int(cu[0]), int(cu[-1])
    return torch.cat([x.new_zeros(lead, H), *outs, x.new_zeros(x.shape[0] - end, H)]), hf


def adjust(logits, context=None, prompt=None, rep=1.0, freq=0.0, pres=0.0, bias_ids=None, bias=None,
           mask=None):
    """Rows of logits (R, V), everything by row."""
    out = logits.double().clone()
    R, V = out.shape
    for r in range(R):
        def of(v):
            return float(v[r]) if torch.is_tensor(v) else v
        row = out[r].tolist()
        if context is not None:
            start = 0 if prompt is None else int(prompt[r])
            ids = context[r].tolist()
            for v in {i for i in ids if 0 <= i < V}:
                x = row[v]
                x = x / of(rep) if x > 0 else x * of(rep)
                c = sum(1 for i, j in enumerate(ids) if j == v and i >= start)
                if c:
                    x = x - of(freq) * c - of(pres)
                row[v] = x
        if bias_ids is not None:
            for i, b in zip(bias_ids[r].tolist(), bias[r].tolist()):
                if 0 <= i < V:
                    row[i] += b
        if mask is not None:
            for v in range(V):
                if not int(mask[r, v // 32]) >> (v % 32) & 1:
                    row[v] = -math.inf
        out[r] = torch.tensor(row, dtype=torch.float64)
    return out


def gradients(outs, wants, leaves):
    """Of outputs that may not hang on any leaf; zero where a leaf is not reached."""
    pairs = [(o, w) for o, w in zip(outs, wants) if o.requires_grad]
    if not pairs:
        return [torch.zeros_like(v) for v in leaves]
    got = torch.autograd.grad([o for o, _ in pairs], leaves, [w for _, w in pairs], allow_unused=True)
    return [torch.zeros_like(v) if g is None else g for g, v in zip(got, leaves)]
