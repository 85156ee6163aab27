"""A gated scan that gives up a wait says so: ltc_scan_status() and
ltc_cuda.device_status(). Waits are given up from the host, by a budget of 0."""

from __future__ import annotations

import os

import pytest
import torch

import ltc_cuda

DEV = "cuda"


@pytest.mark.skipif(not os.path.isfile(ltc_cuda.LIB_PATH), reason="libltc_hip.so not built")
def test_status_without_gpu():
    capi = ltc_cuda.load_capi(ltc_cuda.LIB_PATH)
    if capi.lib.ltc_device_count() == 0:
        assert capi.lib.ltc_scan_status(0) == 3 and "scan status" in capi.last_error()


@pytest.fixture()
def capi():
    c = ltc_cuda._cuda_module.capi
    c.lib.ltc_scan_status(1)
    yield c
    c.lib.ltc_scan_status(1)


class _NoBudget:
    def __init__(self, lib):
        self.lib = lib

    def __enter__(self):
        self.prev = self.lib.ltc_set_cluster_spin_ticks(0)

    def __exit__(self, *exc):
        self.lib.ltc_set_cluster_spin_ticks(self.prev)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,form", [(torch.float32, "blend"), (torch.bfloat16, "decay")])
def test_a_given_up_wait_is_reported(capi, dtype, form, packed):
    x, gate = (torch.randn(1, 700, 40, device=DEV).to(dtype) for _ in range(2))
    gate = -gate.abs()
    cu = torch.tensor([0, 300, 700], dtype=torch.int32, device=DEV) if packed else None
    if packed:
        x, gate = x[0], gate[0]
    x.requires_grad_(True)
    out, _ = ltc_cuda.ltc_gated_scan(x, gate, cu_seqlens=cu, form=form)
    torch.autograd.grad(out, [x], torch.ones_like(out), retain_graph=True)
    ltc_cuda.device_status()  # nothing was given up
    with _NoBudget(capi.lib):
        with torch.no_grad():
            lost, _ = ltc_cuda.ltc_gated_scan(x, gate, cu_seqlens=cu, form=form)
    assert lost.isnan().any()
    capi.device_status(clear=False)  # the other kernels' flag stays down
    assert capi.lib.ltc_scan_status(0) == 3 and "gave up" in capi.last_error()
    with pytest.raises(RuntimeError, match="gated scan.*gave up"):
        ltc_cuda.device_status()
    ltc_cuda.device_status()  # cleared by the call that raised
    with _NoBudget(capi.lib):
        gx, = torch.autograd.grad(out, [x], torch.ones_like(out))
    assert gx.isnan().any()
    assert capi.lib.ltc_scan_status(1) == 3
    assert capi.lib.ltc_scan_status(0) == 0


@pytest.mark.gpu
def test_calls_that_wait_for_nobody_raise_nothing(capi):
    """One tile, tiles that begin with a sequence, tokens of no sequence."""
    with _NoBudget(capi.lib), torch.no_grad():
        for B, T in ((1, 128), (300, 1), (9, 64)):
            x = torch.randn(B, T, 8, device=DEV)
            assert not ltc_cuda.ltc_gated_scan(x, x)[0].isnan().any()
        x = torch.randn(512, 8, device=DEV)
        cu = torch.tensor([0, 128, 256], dtype=torch.int32, device=DEV)
        assert not ltc_cuda.ltc_gated_scan(x, x, cu_seqlens=cu)[0].isnan().any()
    ltc_cuda.device_status()
