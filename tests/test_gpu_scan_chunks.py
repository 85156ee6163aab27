"""Selective scans that are cut into chunks, in all forms that test_chunks of
test_gpu_selective_scan leaves out: more than 16 states, groups (also of more than 64
channels) and types of 16 bits. Checks and tolerances are that file's."""

from __future__ import annotations

import pytest

import test_gpu_selective_scan as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead,cu", [((1, 200), None), ((2, 150), None), ((200,), [0, 60, 60, 61, 130, 190]),
                                     ((170,), [7, 170])])
@pytest.mark.parametrize("H,N,G,dtype,skip,gated,softplus,state", [
    (5, 17, 1, "fp32", True, True, True, True), (6, 24, 2, "bf16", True, False, True, True),
    (130, 32, 2, "fp32", False, True, True, False), (4, 33, 1, "fp16", True, True, False, True),
    (3, 64, 1, "fp32", True, False, True, True), (140, 64, 2, "bf16", True, True, True, True),
    (12, 40, 3, "fp16", False, True, True, True), (140, 16, 2, "bf16", True, True, True, True),
    (6, 5, 3, "fp16", True, False, True, False)])
def test_chunks_of_every_form(lead, cu, H, N, G, dtype, skip, gated, softplus, state):
    S._check(lead, cu, H, N, G, dtype, skip, gated, softplus, state)
