"""The sequence and token operators at their limits on the GPU: tensors of more than 2^31
elements, a wait budget of nothing, states that overlap what is read, empty inputs of the
modules, calls under way on two streams at once."""

from __future__ import annotations

import pytest
import torch

import ltc
import ltc_cuda
from _gpu_common import DEV, _native  # noqa: F401
import _seq_ref as R

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
DEFAULT_TICKS = 20_000_000


@pytest.mark.parametrize("packed", [False, True])
def test_scan_past_32_bits(packed):
    """The last and the first tokens of 2.16e9 elements. Blend gates of normal logits
    shrink a state by exp(-0.8) a token on average: what lies 300 tokens off adds
    nothing that float32 holds."""
    N, H = 1_050_000, 2056
    g = torch.Generator(DEV).manual_seed(7)
    x, gate, go = (torch.randn(N, H, generator=g, device=DEV, dtype=BF16) for _ in range(3))
    x.requires_grad_(True)
    gate.requires_grad_(True)
    if packed:
        cu = torch.tensor([0, N - 450, N], dtype=torch.int32, device=DEV)
        out, hf = ltc_cuda.ltc_gated_scan(x, gate, cu_seqlens=cu)
    else:
        out, hf = ltc_cuda.ltc_gated_scan(x[None], gate[None])
        out = out[0]
    gx, gg = torch.autograd.grad(out, [x, gate], go)
    got = {"out": out.detach(), "gx": gx, "gg": gg}
    n, keep = 400, 100
    for part, rows in ((slice(N - n, N), slice(n - keep, n)), (slice(0, n), slice(0, keep))):
        zero = torch.zeros(1, H)
        val, tol = R.scan(x[part].detach().cpu(), gate[part].detach().cpu(), zero, "blend", [(0, n)],
                          go[part].cpu(), zero)
        for name, t in got.items():
            R.close(t[part][rows].cpu(), val[name][rows], tol[name][rows], f"{name} {part.start}")
        if part.start > 0:
            R.close(hf[-1:].detach().cpu(), val["hf"], tol["hf"], "hf")


def test_step_past_32_bits():
    P, H = 1_050_000, 2056
    state = torch.zeros(P, H, device=DEV)
    rows = [0, P - 1, P - 2]
    g = torch.Generator().manual_seed(3)
    x, gate, h = torch.randn(4, H, generator=g), torch.randn(4, H, generator=g), torch.randn(3, H, generator=g)
    for r, v in zip(rows, h):
        state[r] = v.to(DEV)
    slots = torch.tensor([*rows, -1], dtype=torch.int32, device=DEV)
    out = ltc_cuda.ltc_gated_scan_step(x.to(DEV), gate.to(DEV), state, slots)
    val, tol = R.scan(x[:3], gate[:3], h, "blend", [(i, i + 1) for i in range(3)])
    R.close(out[:3].cpu(), val["out"], tol["out"], "out")
    assert not out[3].any()
    for i, r in enumerate(rows):
        assert torch.equal(state[r], out[i])
    assert not state[1:P - 2].any()


def test_token_operators_past_32_bits():
    N, V, K = 17000, 128256, 9
    g = torch.Generator(DEV).manual_seed(5)
    x = torch.randn(N, V, generator=g, device=DEV, dtype=BF16).requires_grad_(True)
    ids = torch.randint(0, V, (N,), generator=g, device=DEV)
    gp, ge = torch.randn(N, generator=g, device=DEV), torch.randn(N, generator=g, device=DEV)
    logp, ent, top_logp, top_ids = ltc_cuda.ltc_token_logprobs(x, ids, top=3)
    gx, = torch.autograd.grad([logp, ent], [x], [gp, ge])
    t = torch.randn(N, K, generator=g, device=DEV)
    tid = torch.randint(0, V, (N, K), generator=g, device=DEV)
    loss = ltc_cuda.ltc_top_distill(x, t, tid)
    gd, = torch.autograd.grad(loss, [x], [gp])
    for part in (slice(0, 2), slice(N - 3, N)):
        c = x[part].detach().cpu()
        val, tol = R.logprobs(c, ids[part].cpu(), 1.0, 3, gp[part].cpu(), ge[part].cpu())
        for name, got in (("logp", logp), ("ent", ent), ("top_logp", top_logp), ("top_ids", top_ids),
                          ("gx", gx)):
            R.close(got[part].detach().cpu(), val[name], tol.get(name, 0.0), f"{name} {part.start}")
        val, tol = R.distill(c, t[part].cpu(), tid[part].cpu(), 1.0, gp[part].cpu())
        R.close(loss[part].detach().cpu(), val["loss"], tol["loss"], f"loss {part.start}")
        R.close(gd[part].cpu(), val["gx"], tol["gx"], f"gx of the loss {part.start}")


def test_scan_without_a_wait_budget():
    """Every wait given up: NaN where a state would have come from another tile, up to the
    sequence's end (backward: its beginning), everything else as ever."""
    capi = ltc_cuda._cuda_module.capi
    B, T, H = 2, 300, 40
    g = torch.Generator().manual_seed(1)
    x, gate, go = (torch.randn(B, T, H, generator=g).to(DEV) for _ in range(3))
    x.requires_grad_(True)
    want, _ = ltc_cuda.ltc_gated_scan(x, gate)
    want_gx, = torch.autograd.grad(want, [x], [go])
    kept, _ = ltc_cuda.ltc_gated_scan(x, gate)
    assert capi.lib.ltc_set_cluster_spin_ticks(0) == DEFAULT_TICKS
    try:
        with torch.no_grad():
            out, hf = ltc_cuda.ltc_gated_scan(x, gate)
        gx, = torch.autograd.grad(kept, [x], [go])
    finally:
        assert capi.lib.ltc_set_cluster_spin_ticks(DEFAULT_TICKS) == 0
    t = torch.arange(B * T, device=DEV)
    tile = t // 128 * 128
    first, last = t // T * T, t // T * T + T - 1
    lost = tile > first
    lost_b = torch.clamp(tile + 127, max=B * T - 1) < last
    for got, ref, gone in ((out, want, lost), (gx, want_gx, lost_b)):
        got, ref = got.detach().reshape(B * T, H), ref.detach().reshape(B * T, H)
        assert got[gone].isnan().all()
        assert torch.equal(got[~gone], ref[~gone])
    assert hf.isnan().all()
    with torch.no_grad():
        again, _ = ltc_cuda.ltc_gated_scan(x, gate)
    assert torch.equal(again, want)


def test_step_refuses_a_state_it_reads():
    state = torch.zeros(4, 8, device=DEV)
    other = torch.zeros(4, 8, device=DEV)
    with torch.no_grad():
        for x, gate in ((state, other), (other, state), (state[:, :], other)):
            with pytest.raises(RuntimeError, match="memory"):
                ltc_cuda.ltc_gated_scan_step(x, gate, state)
        # apart in one buffer they are fine
        both = torch.zeros(2, 4, 8, device=DEV)
        ltc_cuda.ltc_gated_scan_step(both[0], other, both[1])


@pytest.mark.parametrize("shape", [(2, 0, 3), (0, 4, 3)])
def test_layer_without_tokens(shape):
    m = ltc.LinearTimeConstant(3, 16).to(DEV)
    h0 = torch.randn(shape[0], 16, device=DEV)
    out, (h, _) = m(torch.zeros(shape, device=DEV), (h0, h0))
    assert out.shape == (*shape[:2], 16)
    assert torch.equal(h, h0)
    if shape[0] == 0:
        with torch.no_grad():
            assert m.step(torch.zeros(0, 3, device=DEV), torch.zeros(0, 16, device=DEV)).shape == (0, 16)


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(2)
    x, gate = (torch.randn(2, 5000, 96, generator=g).to(DEV) for _ in range(2))
    logits = torch.randn(6, 50000, generator=g).to(DEV)
    ids = torch.randint(0, 50000, (6,), generator=g).to(DEV)

    def work():
        with torch.no_grad():
            return [*ltc_cuda.ltc_gated_scan(x, gate), *ltc_cuda.ltc_token_logprobs(logits, ids, top=20)]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for res in got:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("N,V,K", [(1030, 20011, 64), (3, 20011, 1000), (1025, 5000, 1), (2, 70, 1024)])
def test_distill_entries_over_segments(N, V, K, dtype):
    """Entries that come several times, at a gradient's segments' edges, missing ones
    between them; the same gradient each time."""
    g = torch.Generator().manual_seed(N + K)
    x, t = torch.randn(N, V, generator=g).to(dtype), torch.randn(N, K, generator=g)
    ids = torch.randint(0, V, (N, K), generator=g)
    edges = torch.tensor([0, 2047, 2048, 4095, 4096, V - 1]).clamp(max=V - 1)
    some = torch.rand(N, K, generator=g)
    ids = torch.where(some < 0.3, edges[torch.randint(0, 6, (N, K), generator=g)], ids)
    ids = torch.where(some > 0.9, -torch.ones_like(ids), ids)
    gl = torch.rand(N, generator=g)
    leaf = x.to(DEV).requires_grad_(True)
    grads = []
    for _ in range(2):
        loss = ltc_cuda.ltc_top_distill(leaf, t.to(DEV), ids.to(DEV), temperature=2.0)
        grads += torch.autograd.grad(loss, [leaf], [gl.to(DEV)])
    assert torch.equal(*grads)
    rows = sorted({0, 1, N - 1})
    val, tol = R.distill(x[rows], t[rows], ids[rows], 2.0, gl[rows])
    R.close(loss.detach().cpu()[rows], val["loss"], tol["loss"], "loss")
    R.close(grads[0].cpu()[rows], val["gx"], tol["gx"], "gx")
