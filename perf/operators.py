"""The sequence and token operators, timed and checked over the range a user meets.

A case is one call: a gated linear recurrence over sequences (forward, or forward
and backward), its step for single tokens, log probabilities of given tokens, or
the distillation loss against a teacher's top logits. With `own` false, `run`
computes it in elementary torch operations in 32 bits; with `own` true, it makes
the calls of ltc_cuda. `exact` is the definition in 64 bits.

Keys of a case:
  op       "scan"      ltc_cuda.ltc_gated_scan
           "step"      ltc_cuda.ltc_gated_scan_step
           "logprobs"  ltc_cuda.ltc_token_logprobs
           "distill"   ltc_cuda.ltc_top_distill
  train    forward and backward (all gradients), else forward without grad
  dtype    of x and of the logits
scan: form ("blend": a = sigmoid(g), h = a h + (1 - a) x; "decay": a = exp(g),
h = a h + x), gate (its dtype), B T H, state (whether one is given), S (0: a
batch of B sequences of T steps; else B = 1 and T tokens of S packed sequences,
one of them empty, some tokens behind the last).
step: form, gate, B H, pool (0: state rows are the batch's; else rows of a pool
that the batch names by slots, some of its rows padding).
logprobs: N V, top (alternatives returned), temperature, masked (share of the
vocabulary at -inf), ignored (share of rows without a token).
distill: N V K, temperature, absent (share of teacher entries missing).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


_kernels = None


def _ops():
    global _kernels
    if _kernels is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "ltc-cuda_amd"))
        import ltc_cuda
        _kernels = ltc_cuda
    return _kernels


def _scan(name, B, T, H, dtype, gate=None, form="blend", state=False, S=0, train=False):
    c = {"op": "scan", "B": B, "T": T, "H": H, "dtype": dtype, "gate": gate or dtype,
         "form": form, "state": state, "S": S, "train": train}
    return {"name": name, **c} if name else c


def _step(name, B, H, dtype, gate=None, form="blend", pool=0):
    c = {"op": "step", "B": B, "H": H, "dtype": dtype, "gate": gate or dtype, "form": form,
         "pool": pool, "train": False}
    return {"name": name, **c} if name else c


def _logprobs(name, N, V, dtype, top=0, temperature=1.0, masked=0.0, ignored=0.0, train=False):
    c = {"op": "logprobs", "N": N, "V": V, "dtype": dtype, "top": top, "temperature": temperature,
         "masked": masked, "ignored": ignored, "train": train}
    return {"name": name, **c} if name else c


def _distill(name, N, V, K, dtype, temperature=1.0, absent=0.0, train=True):
    c = {"op": "distill", "N": N, "V": V, "K": K, "dtype": dtype, "temperature": temperature,
         "absent": absent, "train": train}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One control tick of one stream: latency is all there is.
        _step("step_b1_h64", 1, 64, "fp32"),
        # A decode step of a server: states in a pool, the batch padded.
        _step("step_b256_pool", 256, 2048, "bf16", gate="fp32", form="decay", pool=1024),
        # Training step on the headline's windows (24 of 8 frames), fp32 as the layer.
        _scan("scan_train_b24_t8", 24, 8, 64, "fp32", train=True),
        # Training step of a wide layer on long windows.
        _scan("scan_train_b8_t4096", 8, 4096, 2048, "bf16", train=True),
        # Training step on packed documents of uneven length, odd sizes, decays kept in fp32.
        _scan("scan_train_packed", 1, 30011, 1000, "bf16", gate="fp32", form="decay",
              state=True, S=37, train=True),
        # Reading one very long recording, its state carried on.
        _scan("scan_long_t131072", 1, 131072, 512, "bf16", state=True),
        # Prompts of a few streams before decoding.
        _scan("scan_prompt_b4_t1999", 4, 1999, 320, "fp16"),
        # What a server reports for each decoded token: its log probability and the best 20.
        _logprobs("logprobs_decode_top20", 8, 32000, "bf16", top=20, temperature=0.7),
        # Scoring a text: fp32 logits, a vocabulary whose rows do not align, padding rows.
        _logprobs("logprobs_score_v50021", 2047, 50021, "fp32", top=5, ignored=0.1),
        # Policy-gradient training: log probability and entropy of the taken token, parts of
        # the vocabulary not allowed.
        _logprobs("logprobs_train_v32768", 4096, 32768, "bf16", masked=0.2, ignored=0.05,
                  train=True),
        # Distilling a small head: few entries, some missing.
        _distill("distill_v10007_k8", 300, 10007, 8, "fp32", absent=0.3),
        # Distilling a large vocabulary, the teacher's 64 best stored per token.
        _distill("distill_v65536_k64", 4096, 65536, 64, "bf16", temperature=2.0),
    ]


def draw(rng):
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    kind = rng.choice(["scan", "scan", "scan", "step", "logprobs", "logprobs", "distill"])
    if kind == "scan":
        H = logint(16, 4096)
        n = logint(4, min(131072, (1 << 26) // H))
        gate = rng.choice([dtype, dtype, "fp32"])
        form, state, train = rng.choice(["blend", "decay"]), rng.random() < 0.5, rng.random() < 0.6
        if n > 64 and rng.random() < 0.4:
            return _scan(None, 1, n, H, dtype, gate, form, state, logint(2, min(200, n // 8)), train)
        T = max(1, min(n, logint(1, 16384)))
        return _scan(None, max(1, n // T), T, H, dtype, gate, form, state, 0, train)
    if kind == "step":
        B = logint(1, 1024)
        pool = rng.choice([0, B + logint(1, 2048)])
        return _step(None, B, logint(16, 4096), dtype, rng.choice([dtype, "fp32"]),
                     rng.choice(["blend", "decay"]), pool)
    V = logint(1000, 131072)
    N = logint(1, min(8192, (1 << 27) // V))
    if kind == "logprobs":
        return _logprobs(None, N, V, dtype, rng.choice([0, 0, 1, 5, 20, 32]),
                         rng.choice([1.0, 0.7, 1.3]), rng.choice([0.0, 0.3]),
                         rng.choice([0.0, 0.2]), rng.random() < 0.5)
    return _distill(None, N, V, logint(1, 256), dtype, rng.choice([1.0, 2.0, 4.0]),
                    rng.choice([0.0, 0.25]))


# ----------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _gate(c, g, *shape):
    """Pre-activations around a memory of some tens of steps; logarithms of decays."""
    z = torch.randn(*shape, generator=g, device=DEV) * 1.5 + 2.0
    if c["form"] == "decay":
        z = -torch.nn.functional.softplus(-z)
    return z.to(TYPES[c["gate"]])


def _packed(c, g):
    """Boundaries of S sequences, the second empty, about 1% of the tokens behind the last."""
    S, T = c["S"], c["T"]
    used = T - T // 100
    w = torch.rand(S, generator=g, device=DEV).double() + 0.02
    if S > 2:
        w[1] = 0.0
    cu = torch.zeros(S + 1, dtype=torch.int32, device=DEV)
    cu[1:] = torch.round(torch.cumsum(w, 0) / w.sum() * used).to(torch.int32)
    return cu


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = TYPES[c["dtype"]]
    st = {"case": c}

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def leaf(t):
        return t.requires_grad_(True) if c["train"] else t

    if c["op"] == "scan":
        B, T, H = c["B"], c["T"], c["H"]
        shape = (T, H) if c["S"] else (B, T, H)
        st["x"], st["gate"] = leaf(rand(*shape).to(dt)), leaf(_gate(c, g, *shape))
        st["cu"] = _packed(c, g) if c["S"] else None
        st["state"] = leaf(rand(c["S"] or B, H) * 0.5) if c["state"] else None
        if c["train"]:
            st["go"], st["gh"] = rand(*shape).to(dt), rand(c["S"] or B, H)
    elif c["op"] == "step":
        B, H = c["B"], c["H"]
        st["x"], st["gate"] = rand(B, H).to(dt), _gate(c, g, B, H)
        st["state"] = rand(c["pool"] or B, H) * 0.5
        st["slots"] = None
        if c["pool"]:
            at = torch.randperm(c["pool"], generator=g, device=DEV)[:B].to(torch.int32)
            pad = torch.rand(B, generator=g, device=DEV) < 0.05
            st["slots"] = torch.where(pad, torch.full_like(at, -1), at)
    else:
        N, V = c["N"], c["V"]
        logits = rand(N, V) * 2.0
        if c["op"] == "logprobs":
            ids = torch.randint(0, V, (N,), generator=g, device=DEV)
            if c["masked"]:
                logits[:, torch.rand(V, generator=g, device=DEV) < c["masked"]] = -math.inf
            # taken tokens are likely ones, and allowed
            logits.scatter_(1, ids[:, None], 2.0 + 3.0 * torch.rand(N, 1, generator=g, device=DEV))
            if c["ignored"]:
                ids[torch.rand(N, generator=g, device=DEV) < c["ignored"]] = -100
            st["ids"] = ids
            if c["train"]:
                st["gp"], st["ge"] = rand(N), rand(N) * 0.1
        else:
            K = c["K"]
            hop = 1 + int(torch.randint(0, max(1, V // K), (1,), generator=g, device=DEV))
            first = torch.randint(0, V, (N, 1), generator=g, device=DEV)
            ids = (first + hop * torch.arange(K, device=DEV)) % V
            t = torch.sort(rand(N, K) * 2.0 + 4.0, dim=1, descending=True).values
            logits.scatter_(1, ids, t + rand(N, K))
            if c["absent"]:
                ids[torch.rand(N, K, generator=g, device=DEV) < c["absent"]] = -1
            st["tids"], st["tlogits"] = ids, t.to(dt)
            # the mean over the tokens; a trainer in fp16 scales its loss up
            st["gp"] = torch.rand(N, generator=g, device=DEV) / (1 if c["dtype"] == "fp16" else N)
        st["logits"] = leaf(logits.to(dt))
    return st


# ------------------------------------------------------------------ plain forms


def _bounds(c, cu, T, B):
    """Of B * T tokens laid end to end: which start a sequence, which sequence that is, and
    which tokens lie behind the last."""
    n = T if c["S"] else B * T
    t = torch.arange(n, device=DEV)
    if not c["S"]:
        return t % T == 0, t // T, torch.zeros_like(t, dtype=torch.bool)
    cl = cu.long()
    sid = torch.searchsorted(cl, t, right=True) - 1
    behind = t >= cl[-1]
    sid = sid.clamp(max=c["S"] - 1)
    return (cl[sid] == t) & ~behind, sid, behind


def _doubling(a, b, longest):
    """h_t = a_t h_{t-1} + b_t along dim 0 by doubling; a is 0 where a sequence starts."""
    d = 1
    while d < longest:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        if 2 * d < longest:
            a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _decays(c, g):
    """a and 1 - a, each to its own relative precision."""
    if c["form"] == "blend":
        return torch.sigmoid(g), torch.sigmoid(-g)
    return torch.exp(g), None


def _plain_scan(st):
    c = st["case"]
    x, gate, s0 = st["x"].detach(), st["gate"].detach(), st["state"]
    H, shape = c["H"], x.shape
    B = c["S"] or c["B"]
    start, sid, behind = _bounds(c, st["cu"], c["T"], c["B"])
    xf = x.reshape(-1, H).float()
    a, na = _decays(c, gate.reshape(-1, H).float())
    u = xf if na is None else na * xf
    h0 = torch.zeros(B, H, device=DEV) if s0 is None else s0.detach()
    col = start[:, None]
    b = torch.where(col, u + a * h0[sid], u)
    az = torch.where(col, torch.zeros_like(a), a)
    longest = c["T"]
    h = _doubling(az, b, longest)
    h = torch.where(behind[:, None], torch.zeros_like(h), h)
    # the last step of each sequence; an empty one keeps its state
    if c["S"]:
        lo, hi = st["cu"][:-1].long(), st["cu"][1:].long()
        hf = torch.where((hi > lo)[:, None], h[(hi - 1).clamp(min=0)], h0)
        ends = (hi - 1)[hi > lo]
    else:
        hf = h.view(B, c["T"], H)[:, -1].contiguous()
        ends = torch.arange(1, B + 1, device=DEV) * c["T"] - 1
    out = h.to(x.dtype).view(shape)
    if not c["train"]:
        return [out, hf]
    go = st["go"].reshape(-1, H).float()
    gh = st["gh"][(st["cu"][1:] > st["cu"][:-1])] if c["S"] else st["gh"]
    go = go.clone()
    go[behind] = 0.0
    go.index_add_(0, ends, gh)
    an = torch.cat([az[1:], torch.zeros_like(az[:1])])  # what carries t+1's gradient to t
    d = _doubling(an.flip(0), go.flip(0), longest).flip(0)
    hp = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    hp = torch.where(col, h0[sid], hp)
    if na is None:
        dx, dg = d, d * hp * a
    else:
        dx, dg = d * na, d * (hp - xf) * a * na
    zero = behind[:, None]
    dx, dg = dx.masked_fill(zero, 0.0), dg.masked_fill(zero, 0.0)
    res = [out, hf, dx.to(x.dtype).view(shape), dg.to(gate.dtype).view(shape)]
    if s0 is not None:
        ds = torch.zeros(B, H, device=DEV)
        if c["S"]:  # the state of an empty sequence is its final state
            ds = torch.where((hi > lo)[:, None], ds, st["gh"])
        ds[sid[start]] = (a * d)[start]
        res.append(ds)
    return res


def _plain_step(st):
    c = st["case"]
    x, state, slots = st["x"], st["state"], st["slots"]
    rows = torch.arange(c["B"], device=DEV) if slots is None else slots.long()
    live = (rows >= 0)[:, None]
    a, na = _decays(c, st["gate"].float())
    u = x.float() if na is None else na * x.float()
    h = a * state[rows.clamp(min=0)] + u
    if slots is None:
        state.copy_(h)
    else:
        # padding rows write back what a live row of theirs would: nothing
        keep = rows >= 0
        state[rows[keep]] = h[keep]
    return [torch.where(live, h, torch.zeros_like(h)).to(x.dtype), state]


def _row_stats(z):
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    return m, e, s


def _plain_logprobs(st):
    c = st["case"]
    x, ids = st["logits"].detach(), st["ids"]
    z = x.float() / c["temperature"]
    live = ids >= 0
    at = ids.clamp(min=0)[:, None]
    m, e, s = _row_stats(z)
    lp = z - m - torch.log(s)
    p = e / s
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    ent = -plp.sum(1)
    logp = torch.where(live, lp.gather(1, at)[:, 0], torch.zeros_like(ent))
    res = [logp, torch.where(live, ent, torch.zeros_like(ent))]
    if c["top"]:
        # equal logits by the lower index
        order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :c["top"]]
        res += [lp.gather(1, order), order]
    if c["train"]:
        gp, ge = (torch.where(live, st[k], torch.zeros_like(ent))[:, None] for k in ("gp", "ge"))
        d = -gp * p - ge * (plp + p * ent[:, None])
        d.scatter_add_(1, at, gp)
        res.append((d / c["temperature"]).to(x.dtype))
    return res


def _plain_distill(st):
    c = st["case"]
    x, ids, tau = st["logits"].detach(), st["tids"], c["temperature"]
    m, e, s = _row_stats(x.float() / tau)
    here = ids >= 0
    at = ids.clamp(min=0)
    t = (st["tlogits"].float() / tau).masked_fill(~here, -math.inf)
    some = here.any(1, keepdim=True)
    t = t - torch.where(some, t.max(1, keepdim=True).values, torch.zeros_like(s))
    w = torch.exp(t)
    total = w.sum(1, keepdim=True)
    p = torch.where(some, w / total.clamp(min=1e-30), torch.zeros_like(w))
    logp = torch.where(p > 0, t - torch.log(total.clamp(min=1e-30)), torch.zeros_like(t))
    logq = (x.gather(1, at).float() / tau - m) - torch.log(s)
    loss = tau * tau * torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
    res = [loss]
    if c["train"]:
        d = (e / s) * some.float()
        d.scatter_add_(1, at, -p)
        res.append((d * (tau * st["gp"][:, None])).to(x.dtype))
    return res


# -------------------------------------------------------------------------- run


def _own(st):
    c, k = st["case"], _ops()
    if c["op"] == "scan":
        with torch.set_grad_enabled(c["train"]):
            out, hf = k.ltc_gated_scan(st["x"], st["gate"], st["state"], cu_seqlens=st["cu"],
                                       form=c["form"])
        if not c["train"]:
            return [out, hf]
        leaves = [st["x"], st["gate"]] + ([st["state"]] if c["state"] else [])
        grads = torch.autograd.grad([out, hf], leaves, [st["go"], st["gh"]])
        return [out.detach(), hf.detach(), *grads]
    if c["op"] == "step":
        out = k.ltc_gated_scan_step(st["x"], st["gate"], st["state"], slots=st["slots"],
                                    form=c["form"])
        return [out, st["state"]]
    if c["op"] == "logprobs":
        with torch.set_grad_enabled(c["train"]):
            res = k.ltc_token_logprobs(st["logits"], st["ids"], top=c["top"],
                                       temperature=c["temperature"])
        outs = [t.detach() for t in res]
        if c["train"]:
            outs += torch.autograd.grad(res[:2], [st["logits"]], [st["gp"], st["ge"]])
        return outs
    with torch.set_grad_enabled(c["train"]):
        loss = k.ltc_top_distill(st["logits"], st["tlogits"], st["tids"],
                                 temperature=c["temperature"])
    outs = [loss.detach()]
    if c["train"]:
        outs += torch.autograd.grad([loss], [st["logits"]], [st["gp"]])
    return outs


PLAIN = {"scan": _plain_scan, "step": _plain_step, "logprobs": _plain_logprobs,
         "distill": _plain_distill}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state)


# -------------------------------------------------------- what a pass must do


def work(case):
    """Each input read once, each output written once. Operations of an element, an
    exponential, a logarithm or a division counted as one: 8 of a step forward and 14
    backward; 7 of a logit forward and 8 backward."""
    c = case
    sz = SIZE[c["dtype"]]
    if c["op"] == "scan":
        n, rows = c["B"] * c["T"] * c["H"], (c["S"] or c["B"]) * c["H"]
        gz = SIZE[c["gate"]]
        b = n * (2 * sz + gz) + 4 * rows * (2 if c["state"] else 1)
        if c["train"]:
            b += n * (2 * sz + gz) + 4 * rows * (2 if c["state"] else 1)
        return {"bytes": float(b), "flops": (22.0 if c["train"] else 8.0) * n}
    if c["op"] == "step":
        n = c["B"] * c["H"]
        return {"bytes": float(n * (2 * sz + SIZE[c["gate"]] + 8) + (4 * c["B"] if c["pool"] else 0)),
                "flops": 8.0 * n}
    n = c["N"] * c["V"]
    if c["op"] == "logprobs":
        b = n * sz * (2 if c["train"] else 1) + c["N"] * (16 + 12 * c["top"] + (8 if c["train"] else 0))
    else:
        b = n * sz * 2 + c["N"] * (8 + c["K"] * (8 + sz))
    return {"bytes": float(b), "flops": (15.0 if c["train"] else 7.0) * n}


# ---------------------------------------------------------- definition in 64 bits


def _exact_scan(st):
    c = st["case"]
    x, g = st["x"].detach().double(), st["gate"].detach().double()
    H = c["H"]
    S = c["S"]
    rows = S or c["B"]
    a = 1.0 / (1.0 + torch.exp(-g)) if c["form"] == "blend" else torch.exp(g)
    na = 1.0 / (1.0 + torch.exp(g)) if c["form"] == "blend" else None
    u = x if na is None else na * x
    h0 = torch.zeros(rows, H, device=DEV, dtype=torch.float64) if st["state"] is None \
        else st["state"].detach().double()
    hp, out = torch.zeros_like(x), torch.zeros_like(x)
    hf = h0.clone()
    # packed: (sequence, first token, end); a batch: one run whose steps hold every row
    if S:
        cu = st["cu"].tolist()
        runs = [(s, cu[s], cu[s + 1]) for s in range(S)]
    else:
        runs = [(slice(None), 0, c["T"])]

    def at(v, t):
        return v[t] if S else v[:, t]

    for s, lo, hi in runs:
        h = h0[s]
        for t in range(lo, hi):
            at(hp, t).copy_(h)
            h = torch.addcmul(at(u, t), at(a, t), h)
            at(out, t).copy_(h)
        hf[s] = h
    res = [out, hf]
    if c["train"]:
        d = torch.zeros_like(x)
        ds = torch.zeros_like(h0)
        go, gh = st["go"].double(), st["gh"].double()
        for s, lo, hi in runs:
            carry = gh[s]
            for t in range(hi - 1, lo - 1, -1):
                e = at(go, t) + carry
                at(d, t).copy_(e)
                carry = at(a, t) * e
            ds[s] = carry
        if na is None:
            res += [d, d * hp * a]
        else:
            res += [d * na, d * (hp - x) * a * na]
        if st["state"] is not None:
            res.append(ds)
    return res


def _exact_step(st):
    c = st["case"]
    x, g, state = st["x"].double(), st["gate"].double(), st["state"].double()
    out = torch.zeros_like(x)
    rows = list(range(c["B"])) if st["slots"] is None else st["slots"].tolist()
    for i, r in enumerate(rows):
        if r < 0:
            continue
        if c["form"] == "blend":
            state[r] = (state[r] + torch.exp(-g[i]) * x[i]) / (1.0 + torch.exp(-g[i]))
        else:
            state[r] = torch.exp(g[i]) * state[r] + x[i]
        out[i] = state[r]
    return [out, state]


def _exact_rows(st, each):
    """each(row logits (V,) in 64 bits over tau, row) for blocks of rows."""
    c = st["case"]
    x = st["logits"].detach()
    parts = []
    block = max(1, (1 << 25) // c["V"])
    for r in range(0, c["N"], block):
        sl = slice(r, min(c["N"], r + block))
        z = x[sl].double() / c["temperature"]
        parts.append(each(z, sl, z - torch.logsumexp(z, 1, keepdim=True)))
    return [None if p[0] is None else torch.cat(p) for p in zip(*parts)]


def _exact_logprobs(st):
    c = st["case"]
    ids = st["ids"]

    def each(z, sl, lq):
        n = z.shape[0]
        one = torch.zeros(n, c["V"], device=DEV, dtype=torch.float64)
        live = (ids[sl] >= 0).double()
        one[torch.arange(n, device=DEV), ids[sl].clamp(min=0)] = 1.0
        q = torch.exp(lq)
        fin = torch.where(torch.isinf(lq), torch.zeros_like(lq), lq)
        ent = -(q * fin).sum(1)
        res = [(one * fin).sum(1) * live, ent * live]
        if c["top"]:
            o = torch.argsort(-z, dim=1, stable=True)[:, :c["top"]]
            res += [lq.gather(1, o), o]
        if c["train"]:
            gp = (st["gp"][sl].double() * live)[:, None]
            ge = (st["ge"][sl].double() * live)[:, None]
            res.append((gp * (one - q) - ge * q * (fin + ent[:, None])) / c["temperature"])
        return res

    return _exact_rows(st, each)


def _exact_distill(st):
    c = st["case"]
    tau = c["temperature"]

    def each(z, sl, lq):
        ids = st["tids"][sl]
        t = st["tlogits"][sl].double() / tau
        here = (ids >= 0).double()
        w = torch.exp(t - t.max()) * here
        tot = w.sum(1, keepdim=True)
        p = torch.where(tot > 0, w / torch.where(tot > 0, tot, torch.ones_like(tot)), w)
        lp = torch.log(torch.where(p > 0, p, torch.ones_like(p)))
        loss = tau * tau * (p * (lp - lq.gather(1, ids.clamp(min=0)))).sum(1)
        target = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), p)
        d = torch.exp(lq) * target.sum(1, keepdim=True) - target
        return [loss, tau * st["gp"][sl].double()[:, None] * d]

    res = _exact_rows(st, each)
    return res if c["train"] else res[:1]


EXACT = {"scan": _exact_scan, "step": _exact_step, "logprobs": _exact_logprobs,
         "distill": _exact_distill}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "step":
        st["state"] = st["state"].clone()
    with torch.no_grad():
        return EXACT[case["op"]](st)
