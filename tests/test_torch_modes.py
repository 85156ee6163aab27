"""Forward-mode differentiation and tracing of the torch extension's entry points: errors,
since neither can look into them. The refusals come before the device is looked at, so
the extension itself is called with CPU tensors here."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

import ltc
import ltc_cuda

GPU = pytest.param("cuda", marks=pytest.mark.gpu)


@pytest.fixture(scope="module")
def ext():
    saved = ltc_cuda._torch_ext
    if saved is None:
        ltc_cuda._load_torch_ext()
    mod = ltc_cuda._torch_ext
    ltc_cuda._torch_ext = saved
    if mod is None:
        pytest.skip("torch extension not built (python ltc-cuda_amd/build.py)")
    return mod


def _calls(ext, device):
    """Each entry point as a function of one floating-point input, the others given, and
    that input; one for each input that may carry a tangent."""
    x = torch.randn(2, 3, 4, device=device)
    y, st = x[:, 0].contiguous(), torch.randn(2, 4, device=device)
    ids = torch.zeros(2, 3, dtype=torch.long, device=device)
    D, H = 4, 4
    m = ltc.TrueLiquidTimeConstant(D, H).to(device)
    named = {**dict(m.named_parameters()), **dict(m.named_buffers())}
    leaves = [named[n].detach() for n in ltc_cuda.MODULE_LEAVES]

    def layer(a, i):
        args = [x, st, *leaves]
        args[i] = a
        return ext.module_apply(args[0], args[1], args[2:], 0.1, 2, 1e-8, 1e-5)[0]

    return [
        ("ltc_module_forward", lambda a: layer(a, 0), x),
        ("ltc_module_forward", lambda a: layer(a, 1), st),
        ("ltc_module_forward", lambda a: layer(a, 2), leaves[0]),
        ("ltc_module_forward", lambda a: layer(a, 18), leaves[16]),
        ("ltc_gated_scan", lambda a: ext.gated_scan(a, x, None, None, 0)[0], x),
        ("ltc_gated_scan", lambda a: ext.gated_scan(x, a, st, None, 1)[0], x),
        ("ltc_gated_scan", lambda a: ext.gated_scan(x, x, a, None, 0)[1], st),
        ("ltc_gated_scan_step", lambda a: ext.gated_scan_step(a, y, st, None, 0), y),
        ("ltc_gated_scan_step", lambda a: ext.gated_scan_step(y, a, st, None, 0), y),
        ("ltc_gated_scan_step", lambda a: ext.gated_scan_step(y, y, a, None, 0), st),
        ("ltc_token_logprobs", lambda a: ext.token_logprobs(a, ids, 0, 1.0)[0], x),
        ("ltc_top_distill", lambda a: ext.top_distill(a, x, ids[..., None].expand(2, 3, 4), 1.0), x),
        ("ltc_top_distill", lambda a: ext.top_distill(x, a, ids[..., None].expand(2, 3, 4), 1.0), x),
    ]


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_tangents_are_refused(ext, device):
    for grad in (True, False):
        for name, f, a in _calls(ext, device):
            with torch.set_grad_enabled(grad), fw.dual_level():
                with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode"):
                    f(fw.make_dual(a, torch.ones_like(a)))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_traces_are_refused(ext, device):
    for name, f, a in _calls(ext, device):
        for trace in (torch.jit.trace, lambda g, v: make_fx(g)(v)):
            with torch.no_grad(), pytest.raises(NotImplementedError, match=f"{name} cannot be traced"):
                trace(f, a)


@pytest.mark.gpu
def test_tensors_without_tangents_pass_and_so_does_a_function_with_its_own_rule(ext):
    """h is linear in x: a Function around the scan may give the tangent by itself."""
    x, t, gate = (torch.randn(2, 200, 8, device="cuda") for _ in range(3))

    class Scan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            return ltc_cuda.ltc_gated_scan(v, gate)[0]

        @staticmethod
        def jvp(ctx, tangent):
            return ltc_cuda.ltc_gated_scan(tangent, gate)[0]

    want, want_t = (ltc_cuda.ltc_gated_scan(v, gate)[0] for v in (x, t))
    with fw.dual_level():
        assert torch.equal(ltc_cuda.ltc_gated_scan(x, gate)[0], want)
        out, tangent = fw.unpack_dual(Scan.apply(fw.make_dual(x, t)))
        assert torch.equal(out, want) and torch.equal(tangent, want_t)
