"""Forward-mode differentiation and tracing of the token model's operators: errors, since
neither can look into them. The refusals come before the device is looked at, so the
extension itself is called with CPU tensors here."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from test_torch_modes import GPU, ext  # noqa: F401


def _calls(ext, device):  # noqa: F811
    x = torch.randn(2, 3, 4, device=device)
    w, b, tail = torch.randn(4, 3, device=device), torch.randn(4, device=device), torch.randn(2, 2, 4, device=device)
    A, bc, h = torch.randn(4, 5, device=device), torch.randn(2, 3, 5, device=device), torch.randn(2, 4, 5, device=device)
    y, one = x[:, 0].contiguous(), bc[:, 0].contiguous()
    ids = torch.zeros(2, 3, dtype=torch.long, device=device)
    full = [x, x, A, bc, bc, b, x, b, h]
    step = [y, y, A, one, one, h, b, y, b]

    def scan(i):
        def f(a):
            return ext.selective_scan(*full[:i], a, *full[i + 1:], None, False)[0]
        return f

    def scan_step(i):
        def f(a):
            return ext.selective_scan_step(*step[:i], a, *step[i + 1:], None, False)
        return f

    calls = [("ltc_causal_conv", lambda a: ext.causal_conv(a, w, b, tail, None, 1)[0], x),
             ("ltc_causal_conv", lambda a: ext.causal_conv(x, a, b, tail, None, 1)[0], w),
             ("ltc_causal_conv", lambda a: ext.causal_conv(x, w, a, tail, None, 1)[0], b),
             ("ltc_causal_conv", lambda a: ext.causal_conv(x, w, b, a, None, 1)[0], tail),
             ("ltc_causal_conv_step", lambda a: ext.causal_conv_step(a, w, tail, b, None, 1), y),
             ("ltc_causal_conv_step", lambda a: ext.causal_conv_step(y, w, a, b, None, 1), tail),
             ("ltc_embed", lambda a: ext.embed(a, ids, 1.0), w),
             ("ltc_adjust_logits", lambda a: ext.adjust_logits(a, None, None, None, None, None, 1.0, 0.0, 0.0, None,
                                                               None, None), x)]
    calls += [("ltc_selective_scan", scan(i), v) for i, v in enumerate(full)]
    return calls + [("ltc_selective_scan_step", scan_step(i), v) for i, v in enumerate(step)]


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_tangents_are_refused(ext, device):  # noqa: F811
    for grad in (True, False):
        for name, f, a in _calls(ext, device):
            with torch.set_grad_enabled(grad), fw.dual_level():
                with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode"):
                    f(fw.make_dual(a, torch.ones_like(a)))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_traces_are_refused(ext, device):  # noqa: F811
    for name, f, a in _calls(ext, device):
        for trace in (torch.jit.trace, lambda g, v: make_fx(g)(v)):
            with torch.no_grad(), pytest.raises(NotImplementedError, match=f"{name} cannot be traced"):
                trace(f, a)
