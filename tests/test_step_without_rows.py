"""A step of no rows, with a pool of states: nothing to do, and no error."""

from __future__ import annotations

import os

import pytest
import torch

import ltc
import ltc_cuda


@pytest.mark.skipif(not os.path.isfile(ltc_cuda.LIB_PATH), reason="libltc_hip.so not built")
def test_c_entry():
    f = ltc_cuda.load_capi(ltc_cuda.LIB_PATH).lib.ltc_gated_scan_step
    for slots in (None, 1):
        for P in (0, 1, 40):
            assert f(None, 4, None, 4, 1, 4, slots, 0, 0, 0, 0, 4, P, None, None) == 0
        assert f(None, 4, None, 4, 1, 4, slots, 0, 0, 0, 0, 4, -1, None, None) == 1


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_no_rows_of_a_pool(device):
    pool = torch.randn(7, 5, device=device)
    keep = pool.clone()
    slots = torch.zeros(0, dtype=torch.int32, device=device)
    if device == "cuda":
        x = torch.zeros(0, 5, device=device)
        assert ltc_cuda.ltc_gated_scan_step(x, x, pool, slots).shape == (0, 5)
    m = ltc.LinearTimeConstant(3, 5).to(device)
    assert m.step(torch.zeros(0, 3, device=device), pool, slots).shape == (0, 5)
    assert torch.equal(pool, keep)
