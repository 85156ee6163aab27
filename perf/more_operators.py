"""Operators of a recurrent token model, timed and checked over the range a user meets.

Tokens come in through an embedding, are mixed by a short causal convolution and a
selective state space scan, and what is answered goes through penalties, biases and a
grammar's mask. A case is one call: forward, or forward and backward. With `own`
false, `run` computes it in elementary torch operations in 32 bits; with `own` true, it
makes the calls of ltc_cuda. `exact` is the definition in 64 bits.

Keys of a case:
  op       "conv"      ltc_cuda.ltc_causal_conv
           "convstep"  ltc_cuda.ltc_causal_conv_step
           "ssm"       ltc_cuda.ltc_selective_scan
           "ssmstep"   ltc_cuda.ltc_selective_scan_step
           "embed"     ltc_cuda.ltc_embed
           "adjust"    ltc_cuda.ltc_adjust_logits
  train    forward and backward (all gradients), else forward without grad
  dtype    of activations, of the table and of the logits
conv, ssm: B T H, state (whether one is given), S (0: a batch of B sequences of T steps;
else B = 1 and T tokens of S packed sequences, one of them empty, some tokens behind the
last). conv: K taps, bias, silu, wtype (the weights' dtype). ssm: N states of a channel,
G groups of channels that share B and C, softplus (of the step size, with a bias), skip
(D x is added), gated (times silu(z)).
convstep, ssmstep: B H, pool (0: state rows are the batch's; else rows of a pool that the
batch names by slots, some of its rows padding).
embed: n ids, V H, scale, ignored (share of ids that are not there).
adjust: R rows, V, ctx (tokens before, part of them the prompt), K biases, mask,
per_row (whether each row has its own penalties).
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


def _named(name, c):
    return {"name": name, **c} if name else c


def _conv(name, B, T, H, K, dtype, bias=True, silu=True, wtype=None, state=False, S=0, train=False):
    return _named(name, {"op": "conv", "B": B, "T": T, "H": H, "K": K, "dtype": dtype, "bias": bias,
                         "silu": silu, "wtype": wtype or dtype, "state": state, "S": S, "train": train})


def _convstep(name, B, H, K, dtype, bias=True, silu=True, wtype=None, pool=0):
    return _named(name, {"op": "convstep", "B": B, "H": H, "K": K, "dtype": dtype, "bias": bias,
                         "silu": silu, "wtype": wtype or dtype, "pool": pool, "train": False})


def _ssm(name, B, T, H, N, dtype, G=1, softplus=True, skip=True, gated=True, state=False, S=0,
         train=False):
    return _named(name, {"op": "ssm", "B": B, "T": T, "H": H, "N": N, "G": G, "dtype": dtype,
                         "softplus": softplus, "skip": skip, "gated": gated, "state": state, "S": S,
                         "train": train})


def _ssmstep(name, B, H, N, dtype, G=1, softplus=True, skip=True, gated=True, pool=0):
    return _named(name, {"op": "ssmstep", "B": B, "H": H, "N": N, "G": G, "dtype": dtype,
                         "softplus": softplus, "skip": skip, "gated": gated, "pool": pool,
                         "train": False})


def _embed(name, n, V, H, dtype, scale=1.0, ignored=0.0, train=True):
    return _named(name, {"op": "embed", "n": n, "V": V, "H": H, "dtype": dtype, "scale": scale,
                         "ignored": ignored, "train": train})


def _adjust(name, R, V, dtype, ctx=0, K=0, mask=False, per_row=False):
    return _named(name, {"op": "adjust", "R": R, "V": V, "dtype": dtype, "ctx": ctx, "K": K,
                         "mask": mask, "per_row": per_row, "train": False})


def listed():
    return [
        # Training step of a wide layer on long windows: the convolution before the scan.
        _conv("conv_train_b8_t4096", 8, 4096, 2048, 4, "bf16", train=True),
        # Packed documents of uneven length, rows that do not fill whole lines, a tail carried in.
        _conv("conv_packed_h1000", 1, 30011, 1000, 4, "fp16", state=True, S=37),
        # A decode step of a server: tails in a pool, the batch padded.
        _convstep("convstep_b256_pool", 256, 2048, 4, "bf16", pool=1024),
        # Training step of a wide layer: the scan with all that goes with it.
        _ssm("ssm_train_b8_t2048", 8, 2048, 2048, 16, "bf16", train=True),
        # Training on packed sequences, odd sizes, channels in groups, step sizes as they are.
        _ssm("ssm_train_packed", 1, 5003, 1000, 24, "fp32", G=4, softplus=False, gated=False,
             state=True, S=11, train=True),
        # Reading one long prompt: time is all there is to split.
        _ssm("ssm_prompt_t8192", 1, 8192, 4096, 16, "fp16"),
        # One control tick of one stream: latency is all there is.
        _ssmstep("ssmstep_b1_h64", 1, 64, 16, "fp32", gated=False),
        # A decode step of a server: states in a pool, the batch padded.
        _ssmstep("ssmstep_b256_pool", 256, 2048, 16, "bf16", pool=1024),
        # Training step over a large vocabulary: as few distinct tokens as text has.
        _embed("embed_train_v65536", 32768, 65536, 2048, "bf16", scale=math.sqrt(2048.0)),
        # A short batch of a small vocabulary, padded.
        _embed("embed_train_small", 8 * 17, 10007, 320, "fp32", ignored=0.1),
        # A decode step of one stream: penalties alone.
        _adjust("adjust_b1_v32000", 1, 32000, "fp32", ctx=300),
        # A decode step of a server under grammars: each request with its own penalties.
        _adjust("adjust_b256_v131072", 256, 131072, "bf16", ctx=2048, K=16, mask=True, per_row=True),
    ]


def draw(rng):
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def coin(p):
        return rng.random() < p

    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    kind = rng.choice(["conv", "conv", "convstep", "ssm", "ssm", "ssm", "ssmstep", "embed", "embed",
                       "adjust", "adjust"])
    if kind in ("conv", "ssm"):
        G = rng.choice([1, 1, 1, 2, 4]) if kind == "ssm" else 1
        H = G * max(1, logint(16, 4096) // G)
        N = rng.choice([1, 3, 4, 8, 16, 16, 16, 24, 32, 64]) if kind == "ssm" else 1
        n = logint(4, min(32768, (1 << 26) // H, (1 << 28) // (H * N)))
        state, train = coin(0.5), coin(0.6)
        B, T, S = 1, n, 0
        if n > 64 and coin(0.4):
            S = logint(2, min(200, n // 8))
        else:
            T = max(1, min(n, logint(1, 16384)))
            B = max(1, n // T)
        if kind == "conv":
            return _conv(None, B, T, H, rng.choice([2, 3, 4, 4, 4, 7]), dtype, coin(0.7), coin(0.7),
                         rng.choice([dtype, "fp32"]), state, S, train)
        return _ssm(None, B, T, H, N, dtype, G, coin(0.7), coin(0.7), coin(0.6), state, S, train)
    if kind in ("convstep", "ssmstep"):
        B = logint(1, 512)
        pool = rng.choice([0, B + logint(1, 1024)])
        H = 4 * logint(4, 1024)
        if kind == "convstep":
            return _convstep(None, B, H, rng.choice([2, 4, 4, 7]), dtype, coin(0.7), coin(0.7),
                             rng.choice([dtype, "fp32"]), pool)
        N = rng.choice([1, 4, 8, 16, 16, 24, 64])
        return _ssmstep(None, max(1, min(B, (1 << 23) // (H * N))), H, N, dtype,
                        rng.choice([1, 1, 2, 4]), coin(0.7), coin(0.7), coin(0.6),
                        min(pool, (1 << 25) // (H * N)) if pool and B * H * N < 1 << 23 else 0)
    if kind == "embed":
        V = logint(100, 131072)
        H = logint(8, min(4096, (1 << 27) // V))
        return _embed(None, logint(1, (1 << 26) // H if H > 1024 else 65536), V, H, dtype,
                      rng.choice([1.0, math.sqrt(H)]), rng.choice([0.0, 0.15]), coin(0.8))
    V = logint(1000, 131072)
    return _adjust(None, logint(1, min(512, (1 << 25) // V)), V, dtype,
                   rng.choice([0, logint(1, 4096), logint(1, 4096)]), rng.choice([0, 1, logint(2, 300)]),
                   coin(0.6), coin(0.5))


# ----------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _packed(S, T, g):
    """Boundaries of S sequences, the second empty, about 1% of the tokens behind the last."""
    used = T - T // 100
    w = torch.rand(S, generator=g, device=DEV).double() + 0.02
    if S > 2:
        w[1] = 0.0
    cu = torch.zeros(S + 1, dtype=torch.int32, device=DEV)
    cu[1:] = torch.round(torch.cumsum(w, 0) / w.sum() * used).to(torch.int32)
    return cu


def _slots(B, pool, g):
    at = torch.randperm(pool, generator=g, device=DEV)[:B].to(torch.int32)
    pad = torch.rand(B, generator=g, device=DEV) < 0.05
    return torch.where(pad, torch.full_like(at, -1), at)


def _frequent(V, shape, g):
    """Ids as a text has them: the frequency falls with the id."""
    u = torch.rand(*shape, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp(0, V - 1)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = TYPES[c["dtype"]]
    st = {"case": c}

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def unif(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=g, device=DEV)

    def leaf(t):
        return t.requires_grad_(True) if c["train"] else t

    if c["op"] in ("conv", "convstep"):
        H, K, wt = c["H"], c["K"], TYPES[c["wtype"]]
        st["w"] = leaf(unif(-1.0, 1.0, H, K).to(wt))
        st["bias"] = leaf((rand(H) * 0.2).to(wt)) if c["bias"] else None
        if c["op"] == "convstep":
            st["x"] = rand(c["B"], H).to(dt)
            st["state"] = rand(c["pool"] or c["B"], K - 1, H).to(dt)
            st["slots"] = _slots(c["B"], c["pool"], g) if c["pool"] else None
            return st
        S = c["S"]
        shape = (c["T"], H) if S else (c["B"], c["T"], H)
        st["x"] = leaf(rand(*shape).to(dt))
        st["cu"] = _packed(S, c["T"], g) if S else None
        st["state"] = leaf(rand(S or c["B"], K - 1, H).to(dt)) if c["state"] else None
        if c["train"]:
            st["go"], st["gh"] = rand(*shape).to(dt), rand(S or c["B"], K - 1, H).to(dt)
    elif c["op"] in ("ssm", "ssmstep"):
        H, N, G = c["H"], c["N"], c["G"]
        step = c["op"] == "ssmstep"
        S = 0 if step else c["S"]
        lead = (c["B"],) if step else (c["T"],) if S else (c["B"], c["T"])
        st["x"] = leaf(rand(*lead, H).to(dt))
        # step sizes between a thousandth and some tenths, decays of 1 to N of them
        size = torch.exp(unif(math.log(1e-3), math.log(0.1), H))
        if c["softplus"]:
            st["dbias"] = leaf(size + torch.log(-torch.expm1(-size)))
            st["delta"] = leaf((rand(*lead, H) * 0.7).to(dt))
        else:
            st["dbias"] = None
            st["delta"] = leaf((size * torch.exp(rand(*lead, H) * 0.5)).to(dt))
        st["A"] = leaf(-torch.arange(1, N + 1, device=DEV).float() * torch.exp(0.3 * rand(H, N)))
        grp = (N,) if G == 1 else (G, N)
        st["Bm"], st["Cm"] = leaf(rand(*lead, *grp).to(dt)), leaf(rand(*lead, *grp).to(dt))
        st["D"] = leaf(1.0 + 0.1 * rand(H)) if c["skip"] else None
        st["z"] = leaf(rand(*lead, H).to(dt)) if c["gated"] else None
        if step:
            st["state"] = rand(c["pool"] or c["B"], H, N)
            st["slots"] = _slots(c["B"], c["pool"], g) if c["pool"] else None
            return st
        st["cu"] = _packed(S, c["T"], g) if S else None
        st["state"] = leaf(rand(S or c["B"], H, N)) if c["state"] else None
        if c["train"]:
            st["go"], st["gh"] = rand(*lead, H).to(dt), rand(S or c["B"], H, N)
    elif c["op"] == "embed":
        st["table"] = leaf((rand(c["V"], c["H"]) / math.sqrt(c["H"])).to(dt))
        ids = _frequent(c["V"], (c["n"],), g)
        if c["ignored"]:
            ids[torch.rand(c["n"], generator=g, device=DEV) < c["ignored"]] = -1
        st["ids"] = ids
        if c["train"]:
            st["go"] = rand(c["n"], c["H"]).to(dt)
    else:
        R, V, ctx = c["R"], c["V"], c["ctx"]
        st["logits"] = (rand(R, V) * 3.0).to(dt)
        st["context"] = st["plen"] = st["bias_ids"] = st["bias"] = st["mask"] = None
        if ctx:
            ids = _frequent(V, (R, ctx), g)
            lens = (unif(0.5, 1.0, R) * ctx).round().long()
            st["plen"] = (unif(0.0, 1.0, R) * lens).to(torch.int32)
            st["context"] = torch.where(torch.arange(ctx, device=DEV) < lens[:, None], ids,
                                        torch.full_like(ids, -1))
        if c["K"]:
            first = torch.randint(0, V, (R, 1), generator=g, device=DEV)
            st["bias_ids"] = (first + 7 * torch.arange(c["K"], device=DEV)) % V
            st["bias"] = rand(R, c["K"]) * 2.0
        if c["mask"]:
            st["mask"] = torch.randint(-(1 << 31), 1 << 31, (R, (V + 31) // 32), generator=g, device=DEV,
                                       dtype=torch.int64).to(torch.int32)
        st["rep"], st["freq"], st["pres"] = 1.2, 0.3, 0.4
        if c["per_row"]:
            st["rep"], st["freq"], st["pres"] = unif(1.0, 1.5, R), unif(0.0, 0.5, R), unif(-0.2, 0.5, R)
    return st


# ------------------------------------------------------------------ plain forms


def _bounds(c, cu):
    """Of the tokens laid end to end: (starts of the sequences and the last one's end, the
    sequence of each token, which tokens lie behind the last)."""
    if not c["S"]:
        B, T = c["B"], c["T"]
        t = torch.arange(B * T, device=DEV)
        return torch.arange(B + 1, device=DEV) * T, t // T, torch.zeros_like(t, dtype=torch.bool)
    cl = cu.long()
    t = torch.arange(c["T"], device=DEV)
    sid = (torch.searchsorted(cl, t, right=True) - 1).clamp(max=c["S"] - 1)
    return cl, sid, t >= cl[-1]


def _silu(v):
    s = torch.sigmoid(v)
    return v * s, s * (1.0 + v * (1.0 - s))


def _plain_conv(st):
    c = st["case"]
    x, H, K = st["x"].detach(), c["H"], c["K"]
    w = st["w"].detach().float()
    cl, sid, behind = _bounds(c, st["cu"])
    xf = x.reshape(-1, H).float()
    n, rows = xf.shape[0], c["S"] or c["B"]
    # every sequence with its tail before it
    at = torch.arange(n, device=DEV) + (sid + 1) * (K - 1)
    seq = torch.arange(rows, device=DEV)
    head = ((cl[:-1] + seq * (K - 1))[:, None] + torch.arange(K - 1, device=DEV)).reshape(-1)
    foot = ((cl[1:] + seq * (K - 1))[:, None] + torch.arange(K - 1, device=DEV)).reshape(-1)
    e = torch.zeros(n + rows * (K - 1), H, device=DEV)
    e[at] = xf
    if st["state"] is not None:
        e[head] = st["state"].detach().float().reshape(-1, H)
    pre = torch.zeros(n, H, device=DEV)
    if st["bias"] is not None:
        pre = pre + st["bias"].detach().float()
    for j in range(K):
        pre = pre + w[:, K - 1 - j] * e[at - j]
    val, slope = _silu(pre) if c["silu"] else (pre, None)
    out = val.masked_fill(behind[:, None], 0.0).to(x.dtype).view(x.shape)
    hf = e[foot].to(x.dtype).view(rows, K - 1, H)
    if not c["train"]:
        return [out, hf]
    d = st["go"].reshape(-1, H).float()
    d = (d if slope is None else d * slope).masked_fill(behind[:, None], 0.0)
    dw = torch.stack([(d * e[at - (K - 1 - k)]).sum(0) for k in range(K)], 1)
    de = torch.zeros_like(e)
    # a sequence shorter than the tail hands rows of its head on: the two may meet
    de.index_add_(0, foot, st["gh"].float().reshape(-1, H))
    for j in range(K):
        de[at - j] += w[:, K - 1 - j] * d
    dx = de[at].masked_fill(behind[:, None], 0.0)
    res = [out, hf, dx.to(x.dtype).view(x.shape), dw.to(st["w"].dtype)]
    if st["bias"] is not None:
        res.append(d.sum(0).to(st["bias"].dtype))
    if st["state"] is not None:
        res.append(de[head].to(x.dtype).view(rows, K - 1, H))
    return res


def _plain_convstep(st):
    c = st["case"]
    x, state, slots = st["x"], st["state"], st["slots"]
    rows = torch.arange(c["B"], device=DEV) if slots is None else slots.long()
    keep = rows >= 0
    win = torch.cat([state[rows.clamp(min=0)], x[:, None]], 1)
    pre = (win.float() * st["w"].float().t()).sum(1)
    if st["bias"] is not None:
        pre = pre + st["bias"].float()
    val = _silu(pre)[0] if c["silu"] else pre
    if slots is None:
        state.copy_(win[:, 1:])
    else:
        state[rows[keep]] = win[keep, 1:]
    return [torch.where(keep[:, None], val, torch.zeros_like(val)).to(x.dtype), state]


def _doubling(a, b, longest):
    """h_t = a_t h_{t-1} + b_t along dim 0 by doubling; a is 0 where a sequence starts."""
    d = 1
    while d < longest:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        if 2 * d < longest:
            a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _step_size(st):
    v = st["delta"].detach().float()
    if st["dbias"] is not None:
        v = v + st["dbias"].detach()
    if not st["case"]["softplus"]:
        return v, None
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs())), torch.sigmoid(v)


def _over_groups(t, G):
    """(n, H, N) summed over the channels of each group, as B and C are shaped."""
    n, H, N = t.shape
    t = t.view(n, G, H // G, N).sum(2)
    return t[:, 0] if G == 1 else t


def _per_channel(t, H, G):
    """(n, N) or (n, G, N) -> (n, H or 1, N)."""
    return t[:, None] if G == 1 else t.repeat_interleave(H // G, 1)


def _plain_ssm(st):
    c = st["case"]
    x, H, N, G = st["x"].detach(), c["H"], c["N"], c["G"]
    rows = c["S"] or c["B"]
    cl, sid, behind = _bounds(c, st["cu"])
    xf = x.reshape(-1, H).float()
    n = xf.shape[0]
    grp = (n, N) if G == 1 else (n, G, N)
    bm = _per_channel(st["Bm"].detach().float().reshape(grp), H, G)
    cm = _per_channel(st["Cm"].detach().float().reshape(grp), H, G)
    size, slope = _step_size(st)
    size = size.reshape(-1, H)
    A = st["A"].detach()
    a = torch.exp(size[:, :, None] * A)
    u = (size * xf)[:, :, None] * bm
    start = (cl[sid] == torch.arange(n, device=DEV)) & ~behind
    h0 = torch.zeros(rows, H, N, device=DEV) if st["state"] is None else st["state"].detach()
    first = start.nonzero()[:, 0] if c["S"] else cl[:-1]
    b = u.clone()
    b[first] += a[first] * h0[sid[first]]
    az = a.clone()
    az[first] = 0.0
    h = _doubling(az, b, c["T"])
    del b
    some = (cl[1:] > cl[:-1])[:, None, None]
    hf = torch.where(some, h[(cl[1:] - 1).clamp(min=0)], h0)
    y = (h * cm).sum(2)
    skip = None if st["D"] is None else st["D"].detach()
    if skip is not None:
        y = y + skip * xf
    out = y
    if c["gated"]:
        gate, gslope = _silu(st["z"].detach().reshape(-1, H).float())
        out = y * gate
    hide = behind[:, None]
    out = out.masked_fill(hide, 0.0).to(x.dtype).view(x.shape)
    if not c["train"]:
        return [out, hf]
    go = st["go"].reshape(-1, H).float().masked_fill(hide, 0.0)
    dy = go * gate if c["gated"] else go
    d = dy[:, :, None] * cm
    gh = torch.where(some, st["gh"], torch.zeros_like(st["gh"]))
    d.index_add_(0, (cl[1:] - 1).clamp(min=0), gh)
    an = torch.cat([az[1:], torch.zeros_like(az[:1])])  # what carries t+1's gradient to t
    d = _doubling(an.flip(0), d.flip(0), c["T"]).flip(0)
    del an, az
    hp = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    hp[first] = h0[sid[first]]
    da = d * hp * a  # the gradient of the exponent
    da[behind] = 0.0
    d[behind] = 0.0
    dsx = (d * bm).sum(2)
    dsize = (da * A).sum(2) + dsx * xf
    dx = dsx * size
    if skip is not None:
        dx = dx + skip * dy
    dpre = dsize if slope is None else dsize * slope.reshape(-1, H)
    gshape = st["Bm"].shape
    res = [out, hf, dx.to(x.dtype).view(x.shape), dpre.to(x.dtype).view(x.shape),
           (da * size[:, :, None]).sum(0),
           _over_groups(d * (size * xf)[:, :, None], G).to(x.dtype).view(gshape),
           _over_groups(h * dy[:, :, None], G).to(x.dtype).view(gshape)]
    if skip is not None:
        res.append((dy * xf).sum(0))
    if c["gated"]:
        res.append((go * y * gslope).to(x.dtype).view(x.shape))
    if st["dbias"] is not None:
        res.append(dpre.sum(0))
    if st["state"] is not None:  # the state of an empty sequence is its final state
        ds = torch.where(some, torch.zeros_like(h0), st["gh"])
        ds[sid[first]] = a[first] * d[first]
        res.append(ds)
    return res


def _plain_ssmstep(st):
    c = st["case"]
    x, state, slots, H, G = st["x"], st["state"], st["slots"], c["H"], c["G"]
    rows = torch.arange(c["B"], device=DEV) if slots is None else slots.long()
    keep = rows >= 0
    size, _ = _step_size(st)
    bm, cm = (_per_channel(st[k].float(), H, G) for k in ("Bm", "Cm"))
    xf = x.float()
    h = torch.exp(size[:, :, None] * st["A"]) * state[rows.clamp(min=0)] + (size * xf)[:, :, None] * bm
    y = (h * cm).sum(2)
    if st["D"] is not None:
        y = y + st["D"] * xf
    if c["gated"]:
        y = y * _silu(st["z"].float())[0]
    if slots is None:
        state.copy_(h)
    else:
        state[rows[keep]] = h[keep]
    return [torch.where(keep[:, None], y, torch.zeros_like(y)).to(x.dtype), state]


def _plain_embed(st):
    c = st["case"]
    table, ids = st["table"].detach(), st["ids"]
    live = (ids >= 0)[:, None]
    at = ids.clamp(min=0)
    out = torch.where(live, table[at].float() * c["scale"], torch.zeros(1, device=DEV)).to(table.dtype)
    if not c["train"]:
        return [out]
    g = torch.zeros(c["V"], c["H"], device=DEV)
    g.index_add_(0, at, torch.where(live, st["go"].float(), torch.zeros(1, device=DEV)))
    return [out, (g * c["scale"]).to(table.dtype)]


def _plain_adjust(st):
    c = st["case"]
    x = st["logits"]
    v = x.float()

    def col(p):
        return p[:, None] if torch.is_tensor(p) else p

    if c["ctx"]:
        ids = st["context"]
        there = ids >= 0
        later = there & (torch.arange(c["ctx"], device=DEV) >= st["plen"][:, None])
        at = ids.clamp(min=0)
        seen = torch.zeros_like(v).scatter_add_(1, at, there.float()) > 0
        count = torch.zeros_like(v).scatter_add_(1, at, later.float())
        rep = col(st["rep"])
        v = torch.where(seen, torch.where(v > 0, v / rep, v * rep), v)
        v = v - col(st["freq"]) * count - col(st["pres"]) * (count > 0).float()
    if c["K"]:
        v = v + torch.zeros_like(v).scatter_add_(1, st["bias_ids"], st["bias"])
    if c["mask"]:
        t = torch.arange(c["V"], device=DEV)
        bit = (st["mask"][:, t // 32] >> (t % 32)) & 1
        v = v.masked_fill(bit == 0, -math.inf)
    return [v.to(x.dtype)]


# -------------------------------------------------------------------------- run


def _grads(outs, wants, st, names):
    leaves = [st[k] for k in names if st.get(k) is not None]
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, wants))


def _own(st):
    c, k = st["case"], _ops()
    act = "silu" if c.get("silu") else None
    if c["op"] == "conv":
        with torch.set_grad_enabled(c["train"]):
            out, hf = k.ltc_causal_conv(st["x"], st["w"], st["bias"], state=st["state"],
                                        cu_seqlens=st["cu"], activation=act)
        if not c["train"]:
            return [out, hf]
        return _grads([out, hf], [st["go"], st["gh"]], st, ["x", "w", "bias", "state"])
    if c["op"] == "convstep":
        out = k.ltc_causal_conv_step(st["x"], st["w"], st["state"], bias=st["bias"], slots=st["slots"],
                                     activation=act)
        return [out, st["state"]]
    if c["op"] == "ssm":
        with torch.set_grad_enabled(c["train"]):
            out, hf = k.ltc_selective_scan(st["x"], st["delta"], st["A"], st["Bm"], st["Cm"], D=st["D"],
                                           z=st["z"], delta_bias=st["dbias"], state=st["state"],
                                           cu_seqlens=st["cu"], delta_softplus=c["softplus"])
        if not c["train"]:
            return [out, hf]
        return _grads([out, hf], [st["go"], st["gh"]], st,
                      ["x", "delta", "A", "Bm", "Cm", "D", "z", "dbias", "state"])
    if c["op"] == "ssmstep":
        out = k.ltc_selective_scan_step(st["x"], st["delta"], st["A"], st["Bm"], st["Cm"], st["state"],
                                        D=st["D"], z=st["z"], delta_bias=st["dbias"], slots=st["slots"],
                                        delta_softplus=c["softplus"])
        return [out, st["state"]]
    if c["op"] == "embed":
        with torch.set_grad_enabled(c["train"]):
            out = k.ltc_embed(st["table"], st["ids"], scale=c["scale"])
        return _grads([out], [st["go"]], st, ["table"]) if c["train"] else [out]
    return [k.ltc_adjust_logits(st["logits"], context=st["context"], prompt_lens=st["plen"],
                                repetition=st["rep"], frequency=st["freq"], presence=st["pres"],
                                bias_ids=st["bias_ids"], bias=st["bias"], mask=st["mask"])]


PLAIN = {"conv": _plain_conv, "convstep": _plain_convstep, "ssm": _plain_ssm,
         "ssmstep": _plain_ssmstep, "embed": _plain_embed, "adjust": _plain_adjust}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state)


# -------------------------------------------------------- what a pass must do


def work(case):
    """Each input read once, each output written once. An exponential, a logarithm, a
    division, a product or a sum counts as one: a convolution 2 a tap and 4 for silu
    forward, twice that and 4 a tap backward; a state of the scan 7 forward and 19
    backward; a channel of a token 12 and 20 more."""
    c = case
    sz, op, train = SIZE[c["dtype"]], c["op"], c["train"]
    if op in ("conv", "convstep"):
        n = c["B"] * c.get("T", 1) * c["H"]
        tail = (c["K"] - 1) * c["H"] * sz
        w = SIZE[c["wtype"]] * c["H"] * (c["K"] + (1 if c["bias"] else 0))
        if op == "convstep":
            return {"bytes": float(2 * n * sz + 2 * c["B"] * tail + w),
                    "flops": float(n * (2 * c["K"] + 4))}
        rows = c["S"] or c["B"]
        b = 2 * n * sz + rows * tail * (2 if c["state"] else 1) + w
        if train:
            b += 2 * n * sz + rows * tail * (2 if c["state"] else 1) + w
        return {"bytes": float(b), "flops": float(n * ((6 * c["K"] + 12) if train else 2 * c["K"] + 4))}
    if op in ("ssm", "ssmstep"):
        t = c["B"] * c.get("T", 1)
        n, H, N = t * c["H"], c["H"], c["N"]
        par = 4 * H * (N + (1 if c["skip"] else 0) + (1 if c["softplus"] else 0))
        bc = 2 * t * c["G"] * N * sz
        acts = 4 if c["gated"] else 3
        if op == "ssmstep":
            return {"bytes": float(acts * n * sz + bc + par + 8 * n * N),
                    "flops": float(n * (7 * N + 12))}
        rows = (c["S"] or c["B"]) * H * N * 4
        b = acts * n * sz + bc + par + rows * (2 if c["state"] else 1)
        if train:
            b += acts * n * sz + bc + par + rows * (2 if c["state"] else 1)
        return {"bytes": float(b), "flops": float(n * ((26 * N + 32) if train else 7 * N + 12))}
    if op == "embed":
        n = c["n"] * c["H"]
        # of the table, the rows that the ids name: at most one an id
        b = 8 * c["n"] + sz * (min(c["n"], c["V"]) * c["H"] + n)
        if train:
            b += sz * (n + c["V"] * c["H"])
        return {"bytes": float(b), "flops": float(n * (2 if train else 1))}
    n = c["R"] * c["V"]
    b = 2 * n * sz + c["R"] * (8 * c["ctx"] + 12 * c["K"]) + (n / 8 if c["mask"] else 0)
    return {"bytes": float(b), "flops": float(n + 8 * c["R"] * c["ctx"])}


# ---------------------------------------------------------- definition in 64 bits


def _runs(c, cu):
    """(sequence, first token, end) of each sequence of a flat token axis."""
    if c["S"]:
        cl = cu.tolist()
        return [(s, cl[s], cl[s + 1]) for s in range(c["S"])]
    return [(b, b * c["T"], (b + 1) * c["T"]) for b in range(c["B"])]


def _exact_conv(st):
    c = st["case"]
    H, K = c["H"], c["K"]

    def dbl(t):
        return None if t is None else t.detach().double().requires_grad_(c["train"])

    x, w, bias, state = dbl(st["x"]), dbl(st["w"]), dbl(st["bias"]), dbl(st["state"])
    with torch.set_grad_enabled(c["train"]):
        flat = x.reshape(-1, H)
        outs, tails, end = [], [], 0
        for s, lo, hi in _runs(c, st["cu"]):
            before = x.new_zeros(K - 1, H) if state is None else state[s]
            line = torch.cat([before, flat[lo:hi]])
            y = sum(line[k:k + hi - lo] * w[:, k] for k in range(K))
            if bias is not None:
                y = y + bias
            outs.append(y / (1.0 + torch.exp(-y)) if c["silu"] else y)
            tails.append(line[hi - lo:])
            end = hi
        outs.append(x.new_zeros(flat.shape[0] - end, H))
        out, hf = torch.cat(outs).view(x.shape), torch.stack(tails)
    res = [out.detach(), hf.detach()]
    if c["train"]:
        leaves = [t for t in (x, w, bias, state) if t is not None]
        res += torch.autograd.grad([out, hf], leaves, [st["go"].double(), st["gh"].double()])
    return res


def _exact_convstep(st):
    c = st["case"]
    x, state, w = st["x"].double(), st["state"].double(), st["w"].double()
    out = torch.zeros_like(x)
    rows = list(range(c["B"])) if st["slots"] is None else st["slots"].tolist()
    for i, r in enumerate(rows):
        if r < 0:
            continue
        line = torch.cat([state[r], x[i:i + 1]])
        y = torch.einsum("kh,hk->h", line, w)
        if st["bias"] is not None:
            y = y + st["bias"].double()
        out[i] = y / (1.0 + torch.exp(-y)) if c["silu"] else y
        state[r] = line[1:]
    return [out, state]


def _exact_size(st):
    v = st["delta"].detach().double()
    if st["dbias"] is not None:
        v = v + st["dbias"].detach().double()
    if not st["case"]["softplus"]:
        return v, torch.ones_like(v)
    return torch.logaddexp(v, torch.zeros_like(v)), 1.0 / (1.0 + torch.exp(-v))


def _exact_ssm(st):
    """Step by step; a batch's rows side by side, packed sequences one after the other."""
    c = st["case"]
    H, N, G, S, T = c["H"], c["N"], c["G"], c["S"], c["T"]
    if c["B"] * T * H * N > 1 << 30:
        return None
    rows = S or c["B"]

    def lanes(t, *shape):  # (steps, sequences side by side, ...)
        t = t.detach().double().reshape(1 if S else c["B"], T, *shape)
        return t.transpose(0, 1)

    x, bm, cm = lanes(st["x"], H), lanes(st["Bm"], G, N), lanes(st["Cm"], G, N)
    size, slope = (lanes(t, H) for t in _exact_size(st))
    A = st["A"].detach().double()
    h0 = x.new_zeros(rows, H, N) if st["state"] is None else st["state"].detach().double()
    if S:
        runs = [(slice(s, s + 1), lo, hi) for s, lo, hi in _runs(c, st["cu"])]
    else:
        runs = [(slice(0, rows), 0, T)]

    def wide(t):  # (rows, G, N) -> (rows, H, N)
        return t[:, :, None].expand(-1, -1, H // G, -1).reshape(t.shape[0], H, N)

    def narrow(t):
        return t.reshape(t.shape[0], G, H // G, N).sum(2)

    y, hf = torch.zeros_like(x), h0.clone()
    before = x.new_zeros(T, x.shape[1], H, N) if c["train"] else None
    for s, lo, hi in runs:
        h = h0[s]
        for t in range(lo, hi):
            if before is not None:
                before[t] = h
            h = torch.exp(size[t][..., None] * A) * h + (size[t] * x[t])[..., None] * wide(bm[t])
            y[t] = (h * wide(cm[t])).sum(-1)
        hf[s] = h
    live = x.new_zeros(T, 1, 1)
    for s, lo, hi in runs:
        live[lo:hi] = 1.0
    if st["D"] is not None:
        y = y + st["D"].detach().double() * x * live
    z = None if st["z"] is None else lanes(st["z"], H)

    def back(t):
        return t.transpose(0, 1).reshape(st["x"].shape)

    sig = None if z is None else 1.0 / (1.0 + torch.exp(-z))
    res = [back(y if z is None else y * z * sig), hf]
    if not c["train"]:
        return res
    go, gh = lanes(st["go"], H) * live, st["gh"].double()
    dy = go if z is None else go * z * sig
    dx, dsize = torch.zeros_like(x), torch.zeros_like(x)
    dA, db, dc, ds = torch.zeros_like(A), torch.zeros_like(bm), torch.zeros_like(cm), torch.zeros_like(h0)
    for s, lo, hi in runs:
        carry = gh[s]
        for t in range(hi - 1, lo - 1, -1):
            a, b = torch.exp(size[t][..., None] * A), wide(bm[t])
            u = size[t] * x[t]
            h = a * before[t] + u[..., None] * b
            d = carry + dy[t][..., None] * wide(cm[t])
            dc[t] = narrow(h * dy[t][..., None])
            db[t] = narrow(d * u[..., None])
            carry = a * d
            e = carry * before[t]
            dA += (e * size[t][..., None]).sum(0)
            into = (d * b).sum(-1)
            dsize[t] = (e * A).sum(-1) + into * x[t]
            dx[t] = into * size[t]
        ds[s] = carry
    if st["D"] is not None:
        dx = dx + st["D"].detach().double() * dy
    dpre = dsize * slope
    res += [back(dx), back(dpre), dA, db.transpose(0, 1).reshape(st["Bm"].shape),
            dc.transpose(0, 1).reshape(st["Cm"].shape)]
    if st["D"] is not None:
        res.append((dy * x).sum((0, 1)))
    if z is not None:
        res.append(back(go * y * sig * (1.0 + z * (1.0 - sig))))
    if st["dbias"] is not None:
        res.append(dpre.sum((0, 1)))
    if st["state"] is not None:
        res.append(ds)
    return res


def _exact_ssmstep(st):
    c = st["case"]
    H, N, G = c["H"], c["N"], c["G"]
    state = st["state"].double()
    size, _ = _exact_size(st)
    x, A = st["x"].double(), st["A"].double()
    out = torch.zeros_like(x)
    rows = list(range(c["B"])) if st["slots"] is None else st["slots"].tolist()
    for i, r in enumerate(rows):
        if r < 0:
            continue
        b, k = (st[m][i].double().reshape(G, 1, N).expand(G, H // G, N).reshape(H, N) for m in ("Bm", "Cm"))
        state[r] = torch.exp(size[i][:, None] * A) * state[r] + (size[i] * x[i])[:, None] * b
        y = torch.einsum("hn,hn->h", state[r], k)
        if st["D"] is not None:
            y = y + st["D"].double() * x[i]
        if st["z"] is not None:
            z = st["z"][i].double()
            y = y * z / (1.0 + torch.exp(-z))
        out[i] = y
    return [out, state]


def _exact_embed(st):
    c = st["case"]
    ids, scale = st["ids"], float(c["scale"])
    table = st["table"].detach()
    out = torch.zeros(c["n"], c["H"], dtype=torch.float64, device=DEV)
    live = (ids >= 0).nonzero()[:, 0]
    out[live] = table[ids[live]].double() * scale
    if not c["train"]:
        return [out]
    # tokens in order, runs of equal ids summed by differences of a running sum's ends
    order = torch.argsort(ids[live], stable=True)
    toks, counts = torch.unique_consecutive(ids[live][order], return_counts=True)
    g = torch.zeros(c["V"], c["H"], dtype=torch.float64, device=DEV)
    ends = torch.cumsum(counts, 0)
    run = torch.cumsum(st["go"].double()[live[order]], 0)
    if toks.numel():
        tot = run[ends - 1]
        tot[1:] -= run[ends[:-1] - 1]
        g[toks] = tot * scale
    return [out, g]


def _exact_adjust(st):
    c = st["case"]
    V = c["V"]
    outs = []
    for r in range(c["R"]):
        v = st["logits"][r].double()
        rep, freq, pres = (float(p[r]) if torch.is_tensor(p) else p
                           for p in (st["rep"], st["freq"], st["pres"]))
        if c["ctx"]:
            ids = st["context"][r]
            every = torch.bincount(ids[ids >= 0], minlength=V)
            tail = ids[int(st["plen"][r]):]
            later = torch.bincount(tail[tail >= 0], minlength=V)
            v = torch.where(every > 0, torch.where(v > 0, v / rep, v * rep), v)
            v = v - freq * later.double() - torch.where(later > 0, pres, 0.0)
        if c["K"]:
            for i, b in zip(st["bias_ids"][r].tolist(), st["bias"][r].tolist()):
                v[i] += b
        if c["mask"]:
            bits = ((st["mask"][r][:, None] >> torch.arange(32, device=DEV)) & 1).reshape(-1)[:V]
            v[bits == 0] = -math.inf
        outs.append(v)
    return [torch.stack(outs)]


EXACT = {"conv": _exact_conv, "convstep": _exact_convstep, "ssm": _exact_ssm,
         "ssmstep": _exact_ssmstep, "embed": _exact_embed, "adjust": _exact_adjust}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "conv":
        return _exact_conv(st)
    with torch.no_grad():
        return EXACT[case["op"]](st)
