"""The sensory sums over very many rows: cut into blocks, so that neither the workspace nor
a launch grows past its bounds."""

from __future__ import annotations

import os

import pytest
import torch

import ltc
import ltc_cuda


@pytest.mark.skipif(not os.path.isfile(ltc_cuda.LIB_PATH), reason="libltc_hip.so not built")
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("N,D,H", [
    (0, 3, 4), (1, 3, 4), (192, 129, 64), (32768, 2049, 2048), (131072, 513, 512), (131072, 65, 64),
    (1 << 20, 2, 64), ((1 << 20) + 1, 2, 64), (5000000, 17, 64), (3000, 4096, 4096), (1500, 9000, 4096)])
def test_blocks_cover_the_rows_within_the_bounds(N, D, H, backward):
    lib = ltc_cuda.load_capi(ltc_cuda.LIB_PATH).lib
    size = lib.ltc_sensory_bwd_workspace_bytes if backward else lib.ltc_sensory_fwd_workspace_bytes
    limit = ltc_cuda.SENSORY_ROW_BYTES
    blocks = ltc_cuda._sensory_blocks(N, D, H, backward)
    assert blocks[0][0] == 0 and blocks[-1][1] == N
    assert all(a[1] == b[0] for a, b in zip(blocks, blocks[1:]))
    lengths = [j - i for i, j in blocks]
    assert max(lengths) <= 1 << 20
    if N:
        # equal but for what the division leaves
        assert min(lengths) >= 1 and max(lengths) - min(lengths) < len(blocks)
        # what does not depend on the rows: the images and the gradients' parts, of which
        # 2048 rows have as many as there can be
        most, fixed = max(lengths), size(2048, D, H) - 4 * 2048 * (2 * H + (H // 32 * D if backward else 0))
        assert size(most, D, H) <= max(size(1024, D, H), fixed + limit + (1 << 20))
    if size(N, D, H) <= limit and N <= 1 << 20:
        assert len(blocks) == 1


class _Recorder:
    """The two entry points in plain torch, which note the rows they were given."""

    def __init__(self):
        self.rows = []

    @staticmethod
    def _sums(x, sigma, mu, w, erev):
        c = w * torch.sigmoid(sigma * (x.unsqueeze(-1) - mu))
        return (c * erev).sum(1), c.sum(1)

    def ltc_sensory_fwd(self, x, *params, out=None):
        self.rows.append(x.shape[0])
        res = self._sums(x, *params)
        if out is None:
            return list(res)
        for o, r in zip(out, res):
            o.copy_(r)
        return list(out)

    def ltc_sensory_bwd(self, gn, gd, x, *params, grad_inputs=None):
        self.rows.append(x.shape[0])
        leaves = [t.detach().requires_grad_(True) for t in (x, *params)]
        with torch.enable_grad():
            g = list(torch.autograd.grad(self._sums(*leaves), leaves, [gn, gd]))
        if grad_inputs is not None:
            grad_inputs.copy_(g[0])
            g[0] = grad_inputs
        return g


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("N,D,H", [(2500, 3, 5), (4100, 70, 130)])
def test_blocks_are_the_calls_on_their_rows(monkeypatch, device, N, D, H):
    """The sums and dL/dx of a block are its own call's, the parameters' gradients the
    calls' added in order."""
    if device == "cpu":
        k = _Recorder()
        monkeypatch.setattr(ltc_cuda, "require_kernels", lambda: k)
    else:
        k = ltc_cuda.require_kernels()
    g = torch.Generator().manual_seed(N)
    shapes = [(N, D)] + [(D, H)] * 4
    leaves = [torch.rand(*q, generator=g).to(device).requires_grad_(True) for q in shapes]
    go = [torch.randn(N, H, generator=g).to(device) for _ in range(2)]
    plain = [t.detach() for t in leaves]
    # few rows: one call
    one = torch.autograd.grad(ltc_cuda.ltc_sensory_sums(*leaves), leaves, go)
    for a, b in zip(one, k.ltc_sensory_bwd(*go, *plain)):
        assert torch.equal(a, b)
    monkeypatch.setattr(ltc_cuda, "SENSORY_ROW_BYTES", 1)  # the least block, 1024 rows
    blocks = ltc_cuda._sensory_blocks(N, D, H, True)
    assert len(blocks) == -(-N // 1024)
    if device == "cpu":
        k.rows.clear()
    got = ltc_cuda.ltc_sensory_sums(*leaves)
    ggot = torch.autograd.grad(got, leaves, go)
    if device == "cpu":
        assert k.rows == [j - i for i, j in blocks] * 2
    total = None
    for i, j in blocks:
        for a, b in zip(got, k.ltc_sensory_fwd(plain[0][i:j], *plain[1:])):
            assert torch.equal(a[i:j], b)
        gx, *gp = k.ltc_sensory_bwd(go[0][i:j], go[1][i:j], plain[0][i:j], *plain[1:])
        assert torch.equal(ggot[0][i:j], gx)
        total = gp if total is None else [a + b for a, b in zip(total, gp)]
    for a, b in zip(ggot[1:], total):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_memory_of_a_long_backward_pass():
    """65536 rows of 1024 inputs and neurons: the parts of dL/dx alone would be 9 GB."""
    m = ltc.LinearTimeConstant(1024, 1024).cuda()
    x = torch.randn(1, 65536, 1024, device="cuda", requires_grad=True)
    out, (h, _) = m(x)
    go = torch.ones_like(out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad(out, [x, *m.parameters()], go)
    torch.cuda.synchronize()
    # a block's workspace with its images and parts (16 + 16 bytes a synapse, few parts),
    # and seven tensors of the rows at once (0.27 GB each)
    most = ltc_cuda.SENSORY_ROW_BYTES + 16 * 16 * 1024 * 1088 + 7 * x.numel() * 4
    assert most < 7e9
    assert torch.cuda.max_memory_allocated() - before <= most
    assert all(torch.isfinite(g).all() for g in grads)


@pytest.mark.gpu
def test_more_rows_than_one_grid_holds():
    N = 65536 * 32 + 5
    m = ltc.LinearTimeConstant(2, 4).cuda()
    x = torch.randn(1, N, 2, device="cuda", requires_grad=True)
    out, (h, _) = m(x)
    gx, gw = torch.autograd.grad(out, [x, m.sensory_w], torch.ones_like(out))
    assert torch.equal(h[0], out[0, -1])
    # the last tokens from the state before them, and the gradients of the last ones
    lead = N - 300
    y = x.detach()[:, lead:].clone().requires_grad_(True)
    tail, _ = m(y, (out.detach()[:, lead - 1], None))
    torch.testing.assert_close(tail, out[:, lead:], rtol=1e-5, atol=1e-6)
    gy, = torch.autograd.grad(tail, [y], torch.ones_like(tail))
    torch.testing.assert_close(gy, gx[:, lead:], rtol=1e-4, atol=1e-6)
    assert torch.isfinite(gw).all()
