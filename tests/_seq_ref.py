"""Plain float64 references of the sequence and token operators, with first-order
bounds on what fp32 arithmetic may lose, shared by their tests.

The bounds are derived, not fitted. One step of the recurrence in fp32 makes, per
term, these relative errors in units of 2^-24: the gate's argument times log2(e),
|g| (an absolute error of |g| log2(e) 2^-24 in the exponent of two, times ln 2); the
hardware exponential and reciprocal one unit in the last place each, 2 + 2; the sums
and products around them 1 each, at most 6. For |g| <= 12 that is below 24, and the
bound of a step's own error is UNIT = 24 * 2^-24 of the sum of its terms' absolute
values. Reassociating the products over tiles adds one rounding per composition, fewer
than the steps they replace. Errors pass on through the same decays: E_t = a_t E_{t-1}
+ UNIT * S_t with S the recurrence of absolute values. What is stored in another type
is off by half a step more, finfo(type).eps / 2 of its value, and by half its smallest
subnormal. The hardware exponential gives 0 where the result is below 2^-126, an error of
less than 2^-126 times what it is multiplied with, here a few units: FLUSH = 8 * 2^-126.
"""

from __future__ import annotations

import torch

UNIT = 24 * 2.0 ** -24
FLUSH = 8 * 2.0 ** -126


def gates(g, form):
    """a and 1 - a (decay: 1) in float64."""
    if form == "blend":
        return torch.sigmoid(g), torch.sigmoid(-g)
    return torch.exp(g), torch.ones_like(g)


def scan(x, gate, state, form, runs, go=None, gh=None):
    """Sequences `runs` = [(first, end)] of flat tokens x, gate (N, H), state (S, H).

    Returns ({name: value}, {name: bound}) with out, hf and, when go is given, gx, gg
    and gs. Non-finite values make their bounds meaningless; the values stand.
    """
    x, g, h0 = x.double(), gate.double(), state.double()
    a, na = gates(g, form)
    u = na * x
    out, eo, hp, eh = (torch.zeros_like(x) for _ in range(4))
    hf, ehf = h0.clone(), torch.zeros_like(h0)
    for s, (lo, hi) in enumerate(runs):
        h, S, E = h0[s], h0[s].abs(), torch.zeros_like(h0[s])
        for t in range(lo, hi):
            hp[t], eh[t] = h, E
            h = a[t] * h + u[t]
            S = a[t] * S + u[t].abs()
            E = a[t] * E + UNIT * S
            out[t], eo[t] = h, E
        hf[s], ehf[s] = h, E
    val, tol = {"out": out, "hf": hf}, {"out": eo, "hf": ehf}
    if go is None:
        return val, tol
    go, gh = go.double(), gh.double()
    d, ed = torch.zeros_like(x), torch.zeros_like(x)
    gs, egs = gh.clone(), torch.zeros_like(h0)
    for s, (lo, hi) in enumerate(runs):
        c, S, E = gh[s], gh[s].abs(), torch.zeros_like(gh[s])
        for t in range(hi - 1, lo - 1, -1):
            d[t], ed[t] = go[t] + c, E + UNIT * (go[t].abs() + S)
            c, S, E = a[t] * d[t], a[t] * (go[t].abs() + S), a[t] * ed[t] + UNIT * (a[t] * d[t]).abs()
        gs[s], egs[s] = c, E
    val["gx"], tol["gx"] = na * d, na * ed + UNIT * (na * d).abs()
    if form == "blend":
        k, dif, mag = a * na, hp - x, hp.abs() + x.abs()
    else:
        k, dif, mag = a, hp, hp.abs()
    val["gg"] = d * dif * k
    tol["gg"] = k * (ed * dif.abs() + d.abs() * (eh + UNIT * mag))
    val["gs"], tol["gs"] = gs, egs
    return val, tol


def logprobs(x, ids, temperature, top=0, gp=None, ge=None):
    """Rows x (N, V), ids (N). One row's sum of exponentials is V / 256 additions deep in
    a thread, then 10 levels of joins, each term good to 4 units times its |z|: the
    relative error of S0 is below rel = (V / 256 + 64) 2^-24, where the 64 covers the
    joins, rescalings and the terms' own errors (sum e^z |z| / S0 is at most log V)."""
    z = x.double() / temperature
    n, V = z.shape
    rel = (V / 256 + 64) * 2.0 ** -24
    lq = torch.log_softmax(z, 1)
    q = lq.exp()
    fin = torch.where(q > 0, lq, torch.zeros_like(lq))
    ent = -(q * fin).sum(1)
    live = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1).long()[:, None]
    zero = torch.zeros_like(ent)
    nan = torch.full_like(ent, float("nan"))

    def masked(v):
        return torch.where(ids >= V, nan, torch.where(live, v, zero))

    lp = lq.gather(1, at)[:, 0]
    val = {"logp": masked(lp), "ent": masked(ent)}
    tol = {"logp": rel + 4 * 2.0 ** -24 * lp.abs(), "ent": rel * (1 + ent.abs())}
    if top:
        order = torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
        val["top_logp"], val["top_ids"] = lq.gather(1, order), order
        tol["top_logp"] = rel + 4 * 2.0 ** -24 * val["top_logp"].abs()
    if gp is not None:
        gl = torch.where(live, gp.double(), zero)[:, None]
        gH = torch.where(live, ge.double(), zero)[:, None]
        one = torch.zeros_like(z).scatter_(1, at, 1.0)
        d = (gl * (one - q) - gH * q * (fin + ent[:, None])) / temperature
        mag = q * (gl.abs() + gH.abs() * (fin.abs() + ent[:, None].abs() + 1)) / temperature
        # the relative error of q: that of S0, and that of its exponent
        val["gx"] = torch.where((ids >= V)[:, None], nan[:, None], d)
        tol["gx"] = mag * (2 * rel + 4 * 2.0 ** -24 * fin.abs()) + 4 * 2.0 ** -24 * one * gl.abs() / temperature
    return val, tol


def distill(x, t, ids, temperature, gl=None):
    """Rows x (N, V); teacher logits t and ids (N, K). Bounds as in logprobs, the teacher's
    sum K / 256 additions deep."""
    tau = temperature
    z, tt = x.double() / tau, t.double() / tau
    n, V = z.shape
    rel = (V / 256 + 64) * 2.0 ** -24
    lq = torch.log_softmax(z, 1)
    here = (ids >= 0) & (tt > -float("inf"))
    some = here.any(1, keepdim=True)
    lp = torch.log_softmax(torch.where(here, tt, torch.full_like(tt, -float("inf"))), 1)
    p = torch.where(here & some, lp.exp(), torch.zeros_like(lp))
    at = ids.clamp(0, V - 1).long()
    term = torch.where(p > 0, p * (lp - lq.gather(1, at)), torch.zeros_like(p))
    bad = (ids >= V).any(1)
    nan = float("nan")
    loss = tau * tau * term.sum(1)
    val = {"loss": torch.where(bad, torch.full_like(loss, nan), loss)}
    mag = torch.where(p > 0, p * (lp.abs() + lq.gather(1, at).abs()), torch.zeros_like(p)).sum(1)
    tol = {"loss": tau * tau * (mag + 1) * 2 * rel}
    if gl is not None:
        q = lq.exp() * some
        target = torch.zeros_like(z).scatter_add_(1, at, p)
        g = tau * gl.double()[:, None]
        val["gx"] = torch.where(bad[:, None], torch.full_like(z, nan), g * (q - target))
        fin = torch.where(q > 0, lq, torch.zeros_like(lq)).abs()
        tol["gx"] = g.abs() * (q * (2 * rel + 4 * 2.0 ** -24 * fin) + target * 2 * rel)
    return val, tol


def close(got, val, tol, what):
    """got is within tol of val, and half a step of its type; equal where not finite."""
    val = val.to(got.device).reshape(got.shape)
    if not got.is_floating_point():
        assert torch.equal(got, val), f"{what}: whole values differ"
        return
    info = torch.finfo(got.dtype)
    tol = tol.to(got.device).reshape(got.shape) if torch.is_tensor(tol) else tol
    # a value past the type's range rounds to infinity
    val = torch.where(val.abs() > info.max, torch.copysign(torch.full_like(val, float("inf")), val), val)
    half = info.eps / 2 if got.dtype != torch.float32 else 2.0 ** -24
    lim = tol + half * (val.abs() + tol) + info.tiny * info.eps + FLUSH
    g = got.double()
    fin = torch.isfinite(val)
    assert torch.equal(torch.isnan(g), torch.isnan(val)), f"{what}: NaN in other places"
    same = (g == val) | torch.isnan(val)
    assert bool(same[~fin].all()), f"{what}: infinities differ"
    err = (g - val).abs()
    over = fin & ~(err <= lim)
    assert not bool(over.any()), (
        f"{what}: {int(over.sum())} of {g.numel()} off, worst {float((err / lim)[over].max()):.2f} "
        f"times the bound (error {float(err[over].max()):.3e})")
