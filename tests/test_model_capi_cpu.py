"""C-ABI of the token model's operators without a GPU: sizes, and refusals before anything
is launched. Fake non-NULL addresses: every case fails its checks, or has no work to do."""

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


def _refused(lib, call, cases):
    for kw, what in cases:
        assert call(**kw) in (1, 2), kw
        assert what in lib.last_error(), (kw, lib.last_error())


def test_conv(lib):
    f = lib.lib

    def fwd(x=1, w=1, cu=None, xt=0, wt=0, act=0, B=2, T=3, C=4, K=4, out=1, hf=1):
        return f.ltc_causal_conv_forward(x, 12, 4, w, None, None, cu, xt, wt, act, B, T, C, K, out, hf, None)

    def bwd(x=1, w=1, xt=0, wt=0, act=0, B=2, T=3, C=4, K=4, ws=256, wsb=BIG):
        return f.ltc_causal_conv_backward(x, 12, 4, w, None, None, None, xt, wt, act, B, T, C, K, None, 0, 0,
                                          None, 1, 1, None, None, ws, wsb, None)

    def step(x=1, w=1, state=1, ssp=12, sst=4, slots=None, xt=0, wt=0, act=0, B=2, C=4, K=4, P=2, out=1):
        return f.ltc_causal_conv_step(x, 4, w, None, state, ssp, sst, slots, xt, wt, act, B, C, K, P, out, None)

    sizes = [({"K": 0}, "K <="), ({"K": 9}, "K <="), ({"C": 0}, "C >= 1"), ({"B": -1}, "B >= 0"),
             ({"xt": 3}, "x_type"), ({"xt": 1, "wt": 2}, "weight_type"), ({"act": 2}, "activation"),
             ({"w": None}, "NULL"), ({"x": None}, "NULL")]
    _refused(lib, fwd, sizes + [({"T": -1}, "T >= 0"), ({"B": INT_MAX, "T": 2}, "too large"),
                                ({"out": None}, "NULL"), ({"hf": None}, "state_final")])
    need = f.ltc_causal_conv_bwd_workspace_bytes(0, 2, 3, 4, 4, 0)
    assert need >= 5 * 4 * 4
    _refused(lib, bwd, sizes + [({"ws": None}, "too small"), ({"wsb": need - 1}, "too small"),
                                ({"ws": 264}, "aligned")])
    _refused(lib, step, sizes + [({"P": 3}, "P must"), ({"P": -1, "slots": 1}, "P must"), ({"sst": 3}, "overlap"),
                                 ({"ssp": 11}, "overlap"), ({"state": None}, "NULL"), ({"out": None}, "NULL"),
                                 ({"B": 65536, "P": 65536}, "65535")])
    assert fwd(B=0, T=0, x=None, out=None, hf=None) == 0
    assert step(B=0, P=3, x=None, out=None) == 0
    for bad in ((3, 2, 3, 4, 4, 0), (0, -1, 3, 4, 4, 0), (0, 2, 3, 4, 9, 0), (0, INT_MAX, 3, 4, 4, 0)):
        assert f.ltc_causal_conv_bwd_workspace_bytes(*bad) == -1


def test_selective_scan(lib):
    f = lib.lib

    def args(x, d, A, Bm, Cm, cu, ty, sp, B, T, H, N, G):
        return (x, 12, 4, d, 12, 4, A, Bm, 6, 2, 2, Cm, 6, 2, 2, None, None, 0, 0, None, None, cu, ty, sp, B, T,
                H, N, G)

    def fwd(x=1, d=1, A=1, Bm=1, Cm=1, cu=None, ty=0, B=2, T=3, H=4, N=2, G=1, save=0, out=1, hf=1, saved=None,
            ws=256, wsb=BIG):
        return f.ltc_selective_scan_forward(*args(x, d, A, Bm, Cm, cu, ty, 1, B, T, H, N, G), save, out, hf, saved,
                                            ws, wsb, None)

    def bwd(x=1, d=1, A=1, Bm=1, Cm=1, ty=0, B=2, T=3, H=4, N=2, G=1, saved=1, gz=None, ws=256, wsb=BIG):
        return f.ltc_selective_scan_backward(*args(x, d, A, Bm, Cm, None, ty, 1, B, T, H, N, G), saved, None, 0, 0,
                                             None, 1, 1, 1, 1, 1, None, gz, None, None, ws, wsb, None)

    def step(x=1, d=1, A=1, Bm=1, Cm=1, state=1, ssp=8, slots=None, ty=0, B=2, H=4, N=2, G=1, P=2, out=1):
        return f.ltc_selective_scan_step(x, 4, d, 4, A, Bm, 2, 2, Cm, 2, 2, None, None, 0, None, state, ssp, slots,
                                         ty, 0, B, H, N, G, P, out, None)

    sizes = [({"H": 0}, "H >= 1"), ({"N": 0}, "N >= 1"), ({"N": 65}, "64 states"), ({"G": 3}, "multiple"),
             ({"G": 0}, "G >= 1"), ({"B": -1}, "B >= 0"), ({"ty": 3}, "type"), ({"x": None}, "NULL"),
             ({"d": None}, "NULL"), ({"A": None}, "NULL"), ({"Bm": None}, "NULL"), ({"Cm": None}, "NULL")]
    # long sequences of few channels are cut, and what enters the pieces is worked out
    assert f.ltc_selective_scan_fwd_workspace_bytes(2, 400, 4, 2, 1, 0) > 0
    big = [({"B": INT_MAX - 1, "T": 2}, "too large"), ({"ws": None, "T": 400}, "too small"), ({"ws": 264}, "aligned")]
    _refused(lib, fwd, sizes + big + [({"out": None}, "NULL"), ({"hf": None}, "state_final"),
                                      ({"save": 1}, "saved"), ({"T": -1}, "T >= 0")])
    _refused(lib, bwd, sizes + big + [({"saved": None}, "saved"), ({"gz": 1}, "grad_z")])
    _refused(lib, step, sizes + [({"P": 3}, "P must"), ({"ssp": 7}, "overlap"), ({"state": None}, "NULL"),
                                 ({"out": None}, "NULL"), ({"B": 65536, "P": 65536}, "65535")])
    assert step(B=0, P=3, x=None, d=None, Bm=None, Cm=None, out=None) == 0
    for q in (f.ltc_selective_scan_saved_floats, f.ltc_selective_scan_fwd_workspace_bytes,
              f.ltc_selective_scan_bwd_workspace_bytes):
        assert q(2, 0, 4, 2, 1, 0) >= 0 and q(0, 9, 4, 2, 1, 0) >= 0 and q(3, 100, 4, 2, 1, 1) >= 0
        for bad in ((-1, 3, 4, 2, 1, 0), (1, 3, 4, 65, 1, 0), (1, 3, 4, 2, 3, 0), (INT_MAX, 3, 4, 2, 1, 0)):
            assert q(*bad) == -1, bad
    # a state before every 16th token, of chunks that are whole batches of 16
    assert f.ltc_selective_scan_saved_floats(3, 33, 4096, 2, 1, 0) == 3 * 3 * 4096 * 2
    assert f.ltc_selective_scan_saved_floats(1, 16, 4, 16, 1, 1) == 64


def test_embed(lib):
    f = lib.lib

    def fwd(t=1, ids=1, ty=0, n=3, V=5, H=4, out=1):
        return f.ltc_embed_forward(t, 4, ids, 1, ty, n, V, H, 1.0, out, None)

    def bwd(ids=1, ty=0, n=3, V=5, H=4, go=1, g=1, ws=256, wsb=BIG):
        return f.ltc_embed_backward(ids, 1, ty, n, V, H, 1.0, go, 4, g, ws, wsb, None)

    sizes = [({"n": -1}, "n >= 0"), ({"V": 0}, "V >= 1"), ({"H": 0}, "H >= 1"), ({"ty": 7}, "type"),
             ({"ids": None}, "NULL"), ({"n": INT_MAX}, "too large")]
    _refused(lib, fwd, sizes + [({"t": None}, "NULL"), ({"out": None}, "NULL")])
    need = f.ltc_embed_bwd_workspace_bytes(3, 5, 4)
    _refused(lib, bwd, sizes + [({"go": None}, "NULL"), ({"g": None}, "NULL"), ({"ws": None}, "too small"),
                                ({"wsb": need - 1}, "too small"), ({"ws": 264}, "aligned")])
    assert fwd(n=0, ids=None, out=None) == 0
    assert f.ltc_embed_bwd_workspace_bytes(-1, 5, 4) == -1 and f.ltc_embed_bwd_workspace_bytes(0, 5, 4) == 0


def test_adjust(lib):
    f = lib.lib

    def call(x=1, ctx=None, n=0, rep=1.0, freq=0.0, pres=0.0, ids=None, bias=None, K=0, ty=0, rows=2, V=5, out=1):
        return f.ltc_adjust_logits(x, 5, ctx, 5, 1, n, None, None, None, None, rep, freq, pres, ids, K, 1, bias, K, K,
                                   None, 1, ty, rows, V, out, None)

    inf, nan = float("inf"), float("nan")
    _refused(lib, call, [({"rows": -1}, "R >= 0"), ({"V": 0}, "V >= 1"), ({"n": -1}, "ctx >= 0"), ({"K": 1025}, "K must"),
                         ({"K": -1}, "K must"), ({"ty": -1}, "logits_type"), ({"rep": 0.0}, "repetition"),
                         ({"rep": inf}, "repetition"), ({"rep": nan}, "repetition"), ({"freq": nan}, "frequency"),
                         ({"pres": inf}, "presence"), ({"x": None}, "NULL"), ({"out": None}, "NULL"),
                         ({"n": 3}, "context"), ({"K": 2}, "bias"), ({"rows": 1 << 40}, "too large"),
                         ({"V": INT_MAX}, "too large")])
    assert call(rows=0, x=None, out=None) == 0
