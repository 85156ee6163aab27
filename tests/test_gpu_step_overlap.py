"""ltc_gated_scan_step refuses x and gate that share memory with the states it writes,
however their rows lie, and takes them where rows only lie between one another."""

from __future__ import annotations

import pytest
import torch

import ltc_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _refused(x, gate, state, slots=None):
    with torch.no_grad(), pytest.raises(RuntimeError, match="memory"):
        ltc_cuda.ltc_gated_scan_step(x, gate, state, slots)


def test_rows_of_a_wider_table():
    table = torch.randn(6, 40, device=DEV)
    other = torch.zeros(4, 8, device=DEV)
    state = table[:, 4:12]
    slots = torch.tensor([3, 2, 1, 0], dtype=torch.int32, device=DEV)
    # the states' own rows, in another order; one channel in common; one row of many
    for t in (table[:4, 4:12], table[:4, 11:19], table[2:, :8], table[5:, 4:12].expand(4, 8)):
        _refused(t, other, state, slots)
        _refused(other, t, state, slots)
    _refused(table[0].view(4, 10)[:, :8], other, state, slots)
    # a table of 16-bit values over the same bytes
    half = table.view(torch.bfloat16)[:4, 8:16]
    _refused(half, other.bfloat16(), state, slots)


def test_rows_that_lie_between_are_taken():
    table = torch.randn(6, 40, device=DEV)
    state = table[:, 4:12]
    slots = torch.tensor([3, 2, 1, 5], dtype=torch.int32, device=DEV)
    for x, gate in ((table[:4, 12:20], table[2:, 20:28]), (table[1:5, 30:38], table[:4, 12:20])):
        before = table.clone()
        xs, gs, want = x.clone(), gate.clone(), state.clone()
        with torch.no_grad():
            o = ltc_cuda.ltc_gated_scan_step(xs, gs, want, slots)
            assert torch.equal(ltc_cuda.ltc_gated_scan_step(x, gate, state, slots), o)
        assert torch.equal(state, want)
        before[:, 4:12] = want
        assert torch.equal(table, before)
    # a transposed input is copied first: it may come from anywhere apart from the states
    big = torch.randn(2, 8, 8, device=DEV)
    st = big[0]
    with torch.no_grad():
        want = st.clone()
        o = ltc_cuda.ltc_gated_scan_step(big[1].t().contiguous(), big[1], want)
        assert torch.equal(ltc_cuda.ltc_gated_scan_step(big[1].t(), big[1], st), o)
    assert torch.equal(st, want)
