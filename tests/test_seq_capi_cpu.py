"""C-ABI of the sequence and token operators without a GPU: sizes, and refusals before
anything is launched. Fake non-NULL addresses: every case fails its checks, or has no
work to do."""

from __future__ import annotations

import os

import pytest
import torch  # noqa: F401  (loads torch's HIP runtime first, as in production)

import ltc_cuda

pytestmark = pytest.mark.skipif(not os.path.isfile(ltc_cuda.LIB_PATH),
                                reason="libltc_hip.so not built (python ltc-cuda_amd/build.py)")

BIG = 1 << 40
INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    return ltc_cuda.load_capi(ltc_cuda.LIB_PATH)


def test_scan_sizes(lib):
    f = lib.lib
    for q in (f.ltc_gated_scan_saved_floats, f.ltc_gated_scan_fwd_workspace_bytes,
              f.ltc_gated_scan_bwd_workspace_bytes):
        assert q(0, 5, 8, 0) >= 0 and q(3, 0, 8, 0) >= 0 and q(3, 0, 8, 1) >= 0
        assert q(2, 1000, 64, 0) <= q(4, 1000, 64, 0)
        for bad in ((-1, 5, 8, 0), (1, -5, 8, 0), (1, 5, 0, 0), (1, 5, -1, 1),
                    (INT_MAX, 1, 8, 0), (INT_MAX // 8, INT_MAX, 8, 0)):
            assert q(*bad) == -1, bad
            assert lib.last_error()
    # a state before every 128th token, and a word per packed token
    assert f.ltc_gated_scan_saved_floats(2, 1000, 64, 0) == 16 * 64
    assert f.ltc_gated_scan_saved_floats(2, 1000, 64, 1) == 8 * 64 + 1024


def _fwd(lib, x=1, gate=1, state=None, cu=None, xt=0, gt=0, form=0, B=2, T=3, H=4, save=0, out=1,
         hf=1, saved=None, ws=256, wsb=BIG):
    return lib.lib.ltc_gated_scan_forward(x, 12, 4, gate, 12, 4, state, cu, xt, gt, form, B, T, H, save,
                                          out, hf, saved, ws, wsb, None)


def _bwd(lib, x=1, gate=1, cu=None, xt=0, gt=0, form=0, B=2, T=3, H=4, saved=1, ws=256, wsb=BIG):
    return lib.lib.ltc_gated_scan_backward(x, 12, 4, gate, 12, 4, None, cu, xt, gt, form, B, T, H, saved,
                                           None, 0, 0, None, 1, 1, None, ws, wsb, None)


def test_scan_refusals(lib):
    # sequences longer than a tile hand states on through the workspace
    need = lib.lib.ltc_gated_scan_fwd_workspace_bytes(2, 400, 4, 0)
    assert need > 0 and lib.lib.ltc_gated_scan_fwd_workspace_bytes(2, 3, 4, 0) == 0
    for call in (_fwd, _bwd):
        for kw, what in (({"H": 0}, "H >= 1"), ({"B": -1}, "B >= 0"), ({"T": -2}, "T >= 0"),
                         ({"xt": 3}, "x_type"), ({"xt": -1}, "x_type"), ({"gt": 1}, "gate_type"),
                         ({"xt": 1, "gt": 2}, "gate_type"), ({"form": 2}, "form"), ({"x": None}, "NULL"),
                         ({"gate": None}, "NULL"), ({"ws": 264}, "aligned")):
            assert call(lib, **kw) == 1, (call.__name__, kw)
            assert what in lib.last_error(), (kw, lib.last_error())
        assert call(lib, B=INT_MAX // 8, T=INT_MAX) == 2
    assert _fwd(lib, T=400, wsb=need - 1) == 1 and "too small" in lib.last_error()
    assert _fwd(lib, T=400, ws=None) == 1 and "too small" in lib.last_error()
    assert _bwd(lib, T=400, ws=None) == 1 and "too small" in lib.last_error()
    assert _fwd(lib, out=None) == 1 and "out" in lib.last_error()
    assert _fwd(lib, hf=None) == 1 and "state_final" in lib.last_error()
    assert _fwd(lib, save=1) == 1 and "saved" in lib.last_error()
    assert _bwd(lib, saved=None) == 1 and "saved" in lib.last_error()


def test_step_refusals(lib):
    def call(x=1, gate=1, state=1, ssp=4, slots=None, xt=0, gt=0, form=0, B=2, H=4, P=2, out=1):
        return lib.lib.ltc_gated_scan_step(x, 4, gate, 4, state, ssp, slots, xt, gt, form, B, H, P, out, None)

    for kw, what in (({"P": 3}, "P must"), ({"P": -1, "slots": 1}, "P must"), ({"ssp": 3}, "overlap"),
                     ({"state": None}, "NULL"), ({"out": None}, "NULL"), ({"x": None}, "NULL"),
                     ({"H": 0}, "H >= 1"), ({"form": -1}, "form"), ({"gt": 1}, "gate_type")):
        assert call(**kw) == 1, kw
        assert what in lib.last_error(), (kw, lib.last_error())
    assert call(B=70000, P=70000) == 2
    assert call(B=0, P=0) == 0


def test_token_sizes(lib):
    f = lib.lib
    assert f.ltc_token_logprobs_workspace_bytes(0, 9, 0, 0) == 0
    assert f.ltc_top_distill_workspace_bytes(0, 9, 0) == 0
    assert f.ltc_token_logprobs_workspace_bytes(100000, 50000, 20, 1) == 0
    few = f.ltc_token_logprobs_workspace_bytes(1, 131072, 0, 1)
    assert 0 < few < f.ltc_token_logprobs_workspace_bytes(1, 131072, 20, 1)
    for bad in ((-1, 9, 0, 0), (4, 0, 0, 0), (4, 9, 10, 0), (4, 90, 33, 0), (4, 9, -1, 0), (4, 9, 0, 3),
                (1 << 33, 9, 0, 0), (1, INT_MAX, 0, 0)):
        assert f.ltc_token_logprobs_workspace_bytes(*bad) == -1, bad
    assert f.ltc_top_distill_workspace_bytes(4, 0, 0) == -1


def test_token_refusals(lib):
    f = lib.lib

    def fwd(x=1, ids=1, ty=0, N=2, V=9, top=0, tau=1.0, logp=1, tl=None, ti=None, ws=None, wsb=0):
        return f.ltc_token_logprobs_forward(x, 9, ids, 1, ty, N, V, top, tau, logp, None, tl, ti, None, ws,
                                            wsb, None)

    def bwd(x=1, ids=1, ty=0, N=2, V=9, tau=1.0, stats=1, gx=1):
        return f.ltc_token_logprobs_backward(x, 9, ids, 1, ty, N, V, tau, stats, None, 0, None, 0, gx, None)

    for call in (fwd, bwd):
        for kw, what in (({"N": -1}, "N >= 0"), ({"V": 0}, "V >= 1"), ({"ty": 7}, "logits_type"),
                         ({"tau": 0.0}, "temperature"), ({"tau": -1.0}, "temperature"),
                         ({"tau": float("nan")}, "temperature"), ({"tau": float("inf")}, "temperature"),
                         ({"tau": 1e-45}, "temperature"), ({"x": None}, "NULL"), ({"ids": None}, "NULL")):
            assert call(**kw) == 1, (call.__name__, kw)
            assert what in lib.last_error(), (kw, lib.last_error())
        assert call(N=1 << 33) == 2 and call(V=INT_MAX) == 2
        assert call(N=0) == 0
    assert fwd(top=1) == 1 and "top_logp" in lib.last_error()
    assert fwd(top=33, V=99) == 1 and "top" in lib.last_error()
    assert fwd(logp=None) == 1
    assert fwd(N=1, V=131072) == 1 and "workspace too small" in lib.last_error()
    assert fwd(N=1, V=131072, ws=8, wsb=BIG) == 1 and "aligned" in lib.last_error()
    assert bwd(stats=None) == 1 and bwd(gx=None) == 1

    def dfw(x=1, t=1, ids=1, ty=0, tt=0, N=2, V=9, K=3, tau=1.0, loss=1, ws=None, wsb=0):
        return f.ltc_top_distill_forward(x, 9, t, 3, ids, 3, 1, ty, tt, N, V, K, tau, loss, None, ws, wsb,
                                         None)

    def dbw(x=1, t=1, ids=1, ty=0, tt=0, N=2, V=9, K=3, tau=1.0, stats=1, gl=1, gx=1):
        return f.ltc_top_distill_backward(x, 9, t, 3, ids, 3, 1, ty, tt, N, V, K, tau, stats, gl, 1, gx, None)

    for call in (dfw, dbw):
        for kw, what in (({"K": 0}, "K must"), ({"K": 1025}, "K must"), ({"tt": 5}, "teacher_type"),
                         ({"ty": 5}, "logits_type"), ({"tau": 0.0}, "temperature"), ({"t": None}, "NULL"),
                         ({"x": None}, "NULL"), ({"ids": None}, "NULL")):
            assert call(**kw) == 1, (call.__name__, kw)
            assert what in lib.last_error(), (kw, lib.last_error())
        assert call(N=0) == 0
    assert dfw(loss=None) == 1 and dbw(stats=None) == 1 and dbw(gl=None) == 1 and dbw(gx=None) == 1
    assert dfw(N=1, V=131072) == 1 and "workspace too small" in lib.last_error()
