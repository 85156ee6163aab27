"""Adjusted logits against the definition, row by row in 64 bits.

Tolerances: a division or product, a multiply-add, a subtraction and a sum of K biases in
float32, each off by half a step of 2^-24 of the largest size met (logit, penalties and
biases together), K + 4 of them, and half a step of the logits' type."""

from __future__ import annotations

import math

import pytest
import torch

import _model_ref as R
import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _close(got, want, size, dtype, K):
    got = got.cpu().double()
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[want.isinf()], want[want.isinf()])
    fin = want.isfinite()
    err = (K + 4) * U * size
    tol = err + R.half_step(dtype) * (want.abs() + err) + torch.finfo(R.TYPES[dtype]).tiny
    assert bool(((got - want).abs() <= tol)[fin].all())


def _run(Rn, V, dtype, ctx=0, prompt=False, K=0, mask=False, per_row=False, ids=torch.int64, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(Rn, V, generator=g) * 3).to(R.TYPES[dtype])
    kw = {}
    if ctx:
        kw["context"] = torch.randint(-3, min(V, 40) + 2, (Rn, ctx), generator=g).to(ids)
        if prompt:
            kw["prompt"] = torch.randint(0, ctx + 2, (Rn,), generator=g, dtype=torch.int32)
    if K:
        kw["bias_ids"] = torch.randint(-2, V + 2, (Rn, K), generator=g).to(ids)
        kw["bias_ids"][:, K // 2:] = kw["bias_ids"][:, :K - K // 2].clone()  # named twice
        kw["bias"] = torch.randn(Rn, K, generator=g) * 2
    if mask:
        kw["mask"] = torch.randint(-(1 << 31), 1 << 31, (Rn, (V + 31) // 32), generator=g).to(torch.int32)
    pen = (1.3, 0.2, 0.5)
    if per_row:
        pen = tuple(torch.rand(Rn, generator=g) + a for a in (0.5, -0.3, -0.3))
    want = R.adjust(x, kw.get("context"), kw.get("prompt"), *pen, kw.get("bias_ids"), kw.get("bias"),
                    kw.get("mask"))
    dev = {k: v.to(DEV) for k, v in kw.items()}
    if "prompt" in dev:
        dev["prompt_lens"] = dev.pop("prompt")
    rep, freq, pres = (p.to(DEV) if torch.is_tensor(p) else p for p in pen)
    got = ltc_cuda.ltc_adjust_logits(x.to(DEV), repetition=rep, frequency=freq, presence=pres, **dev)
    assert got.dtype == x.dtype and got.shape == x.shape
    size = x.double().abs() * 2 + 2 * ctx + 1 + (kw["bias"].abs().sum(1, keepdim=True).double() if K else 0)
    _close(got, want, size, dtype, K)
    return x, dev, got


@pytest.mark.parametrize("Rn,V", [(1, 1), (1, 5), (3, 31), (2, 32), (2, 33), (1, 1023), (2, 1024), (2, 1025),
                                  (0, 40), (1, 2500)])
@pytest.mark.parametrize("dtype,ctx,prompt,K,mask,per_row,ids", [
    ("fp32", 0, False, 0, False, False, torch.int64), ("fp32", 20, True, 6, True, True, torch.int64),
    ("bf16", 300, False, 0, False, False, torch.int32), ("fp16", 1, True, 3, False, True, torch.int32),
    ("bf16", 0, False, 1, True, False, torch.int64), ("fp16", 70, True, 0, True, False, torch.int64)])
def test_against_definition(Rn, V, dtype, ctx, prompt, K, mask, per_row, ids):
    _run(Rn, V, dtype, ctx, prompt, K, mask, per_row, ids)


def test_segments_of_every_length():
    """So many rows that a workgroup's share of a row grows; and the largest list of biases."""
    for rows, V in ((300, 9000), (700, 9000), (1500, 17000)):
        x = torch.randn(rows, V, device=DEV)
        ids = torch.randint(0, V, (rows, 50), device=DEV)
        got = ltc_cuda.ltc_adjust_logits(x, ids, repetition=2.0, frequency=0.5)
        count = torch.zeros(rows, V, device=DEV).scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))
        want = torch.where(count > 0, torch.where(x > 0, x / 2, x * 2), x) - 0.5 * count
        assert float((got - want).abs().max()) <= 4 * U * 40
        assert torch.equal(got[count == 0], x[count == 0])
    _run(2, 3000, "fp32", 10, True, 1024, True, True)


def test_values_that_are_not_numbers():
    x = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -0.0, torch.finfo(torch.float32).min, 2.0, math.nan]],
                     device=DEV)
    ctx = torch.arange(7, device=DEV)[None]
    got = ltc_cuda.ltc_adjust_logits(x, ctx, repetition=2.0, presence=1.0)[0].cpu()
    assert got[0] == math.inf and got[1] == -math.inf and got[2].isnan() and got[3] == -1 and got[4] == -1
    assert got[5] == -math.inf and got[6] == 0 and got[7].isnan()
    mask = torch.tensor([[0b01100000]], dtype=torch.int32, device=DEV)
    got = ltc_cuda.ltc_adjust_logits(x, mask=mask, bias_ids=torch.tensor([[2, 6]], device=DEV),
                                     bias=torch.tensor([[math.inf, 1.0]], device=DEV))[0].cpu()
    assert bool((got[[0, 1, 2, 3, 4, 7]] == -math.inf).all()) and got[6] == 3
    none = ltc_cuda.ltc_adjust_logits(x, mask=torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    assert bool((none == -math.inf).all())


def test_shared_rows_shapes_and_layouts():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 4, 100, generator=g).to(DEV)
    ctx = torch.randint(0, 100, (20,), generator=g).to(DEV)
    mask = torch.randint(-(1 << 31), 1 << 31, (4,), generator=g).to(torch.int32).to(DEV)
    ids, b = torch.tensor([5, 90], device=DEV), torch.tensor([1.0, -2.0], device=DEV)
    rep = (torch.rand(3, 4, generator=g) + 0.5).to(DEV)
    one = ltc_cuda.ltc_adjust_logits(x, ctx, repetition=rep, bias_ids=ids, bias=b, mask=mask)
    many = ltc_cuda.ltc_adjust_logits(x, ctx.expand(3, 4, 20), repetition=rep, bias_ids=ids.expand(3, 4, 2).contiguous(),
                                      bias=b.expand(3, 4, 2), mask=mask.expand(3, 4, 4))
    assert torch.equal(one, many)
    big = torch.randn(3, 4, 140, generator=g).to(DEV)
    big[..., :100] = x
    assert torch.equal(ltc_cuda.ltc_adjust_logits(big[..., :100], ctx, repetition=1.5),
                       ltc_cuda.ltc_adjust_logits(x, ctx, repetition=1.5))
    tr = x.transpose(0, 1)
    assert torch.equal(ltc_cuda.ltc_adjust_logits(tr, ctx, frequency=1.0).transpose(0, 1),
                       ltc_cuda.ltc_adjust_logits(x, ctx, frequency=1.0))
    flat = ltc_cuda.ltc_adjust_logits(x[0, 0], ctx, repetition=rep[0, 0], bias_ids=ids, bias=b, mask=mask)
    assert torch.equal(flat, one[0, 0])
    assert torch.equal(ltc_cuda.ltc_adjust_logits(x), x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ltc_cuda.ltc_adjust_logits(x, ctx, repetition=rep, bias_ids=ids, bias=b, mask=mask)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, one)


def test_ids_of_any_value():
    x = torch.randn(1, 50, device=DEV)
    wild = torch.tensor([[-(1 << 63), (1 << 63) - 1, 1 << 32, -1, 50, 49]], device=DEV)
    got = ltc_cuda.ltc_adjust_logits(x, wild, presence=1.0, bias_ids=wild, bias=torch.ones(1, 6, device=DEV))
    want = x.clone()
    want[0, 49] = (want[0, 49] - 1.0) + 1.0
    assert torch.equal(got, want)


def test_refusals():
    x = torch.randn(2, 40, device=DEV)
    ids = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    f = ltc_cuda.ltc_adjust_logits

    def wrong(exc, *a, **kw):
        with pytest.raises(exc):
            f(*a, **kw)

    wrong(ValueError, x.cpu(), ids.cpu())
    wrong(TypeError, x.double())
    wrong(ValueError, x, ids.cpu())
    wrong(TypeError, x, ids.float())
    wrong(ValueError, x, ids[:1])
    for r in (0.0, -1.0, math.inf, math.nan):
        wrong(ValueError, x, ids, repetition=r)
    wrong(ValueError, x, ids, frequency=math.inf)
    wrong(ValueError, x, ids, presence=math.nan)
    wrong(ValueError, x, ids, repetition=torch.ones(3, device=DEV))
    wrong(TypeError, x, ids, repetition=torch.ones(2, device=DEV).half())
    wrong(ValueError, x, prompt_lens=torch.zeros(2, dtype=torch.int32, device=DEV))
    wrong(TypeError, x, ids, prompt_lens=torch.zeros(2, dtype=torch.int64, device=DEV))
    wrong(ValueError, x, ids, prompt_lens=torch.zeros(3, dtype=torch.int32, device=DEV))
    wrong(ValueError, x, bias_ids=ids)
    wrong(ValueError, x, bias_ids=ids, bias=torch.zeros(2, 4, device=DEV))
    wrong(TypeError, x, bias_ids=ids, bias=torch.zeros(2, 3, device=DEV).half())
    wrong(ValueError, x, bias_ids=torch.zeros(2, 1025, dtype=torch.int64, device=DEV),
          bias=torch.zeros(2, 1025, device=DEV))
    wrong(ValueError, x, mask=torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    wrong(TypeError, x, mask=torch.zeros(2, 2, dtype=torch.int64, device=DEV))
    wrong(RuntimeError, x.requires_grad_(True), ids)
