"""The least temperature of the token operators: its scale of the logits has to be finite,
or equal logits would become 0 times an infinity. No GPU: nothing is launched."""

from __future__ import annotations

import os

import pytest
import torch  # noqa: F401  (loads torch's HIP runtime first, as in production)

import ltc_cuda

pytestmark = pytest.mark.skipif(not os.path.isfile(ltc_cuda.LIB_PATH),
                                reason="libltc_hip.so not built (python ltc-cuda_amd/build.py)")


@pytest.mark.parametrize("tau,taken", [(1e-30, True), (4.3e-39, True), (4.2e-39, False), (3e-39, False)])
def test_least_temperature(tau, taken):
    capi = ltc_cuda.load_capi(ltc_cuda.LIB_PATH)
    f = capi.lib
    for N in (0, 2):  # without rows nothing runs, with them the next check fails
        calls = [
            f.ltc_token_logprobs_forward(None, 9, 1, 1, 0, N, 9, 0, tau, 1, None, None, None, None, None, 0,
                                         None),
            f.ltc_token_logprobs_backward(None, 9, 1, 1, 0, N, 9, tau, 1, None, 0, None, 0, 1, None),
            f.ltc_top_distill_forward(None, 9, 1, 3, 1, 3, 1, 0, 0, N, 9, 3, tau, 1, None, None, 0, None),
            f.ltc_top_distill_backward(None, 9, 1, 3, 1, 3, 1, 0, 0, N, 9, 3, tau, 1, 1, 1, 1, None)]
        assert calls == [0 if taken and N == 0 else 1] * 4
        if N or not taken:
            assert ("NULL" if taken else "temperature") in capi.last_error()
