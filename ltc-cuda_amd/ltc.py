"""Liquid Time-Constant layer with an MI355X-native fused ODE solver (drop-in for ltc.py).

Same public surface as the reference module (ltc.py:109-349):
`TrueLiquidTimeConstant(input_dim, hidden_dim=64, dt=1/30, ode_unfolds=6,
sparsity=0.5, sensory_sparsity=0.5, input_mapping="affine", epsilon=1e-8)`,
`forward(x_seq, h0=None) -> (outputs, (h, h))`, the same parameter and buffer
names (so state_dicts load across), the same RNG consumption order at init (so
a seed builds the same tensors), the eval-mode transform cache, the
`_force_torchscript` switch, the `W_rec` / `fused_euler_step` shims and the
`TemporalLTC` alias.

Dispatch. fp32 tensors on a HIP device go to the fused kernels in
libltc_hip.so. In training mode the whole layer (LayerNorm, affine, softplus
transforms and the ODE loop, and their backward) is one library call each way
(`ltc_cuda.ltc_module_forward`). In eval mode the reference's transform cache
applies (ltc.py:270-288) and the cached boundary tensors go through
`ltc_cuda.ltc_cuda_forward`, as in the reference. If the library is not
loaded, the call raises: on a GPU the fused path is never swapped for another
one behind the caller's back. CPU tensors, non-fp32 tensors and an explicit
`module._force_torchscript = True` use the TorchScript loop below, which is
this module's own CPU implementation of the same equations (the reference
does the same, ltc.py:293-323).

Beyond the reference: `LinearTimeConstant`, the layer without recurrent synapses, whose
time axis is parallel; `TokenEmbedding`, `SelectiveTimeConstant` and `TokenReadout`, which
make a model over tokens: rows of a table in, a layer whose time constants the input
selects, token scores, losses and adjusted scores out.
"""

from __future__ import annotations

import logging

import torch
import torch.nn as nn
import torch.nn.functional as F

import ltc_cuda
from ltc_cuda import _HAS_CUDA_KERNELS, ltc_cuda_forward  # noqa: F401  (reference import surface)

logger = logging.getLogger(__name__)


@torch.jit.script
def _ltc_ode_step_jit(
    inputs: torch.Tensor,        # (B, D)
    state: torch.Tensor,         # (B, H)
    w_pos: torch.Tensor,         # (H, H) softplus(w) * sparsity_mask
    w_erev: torch.Tensor,        # (H, H) w_pos * erev
    mu: torch.Tensor,            # (H, H)
    sigma: torch.Tensor,         # (H, H)
    sensory_mu: torch.Tensor,    # (D, H)
    sensory_sigma: torch.Tensor, # (D, H)
    sensory_erev: torch.Tensor,  # (D, H)
    sensory_w_pos: torch.Tensor, # (D, H) softplus(sensory_w) * mask
    cm_t: torch.Tensor,          # (H,)
    gleak_pos: torch.Tensor,     # (H,)
    vleak: torch.Tensor,         # (H,)
    ode_unfolds: int,
    epsilon: float,
) -> torch.Tensor:
    """One time step: sensory conductances, then `ode_unfolds` implicit-Euler updates.

    Reductions run over dim 1: inputs d for the sensory (B, D, H) product and
    presynaptic i for the recurrent (B, H, H) product (ltc.py:42-63).
    """
    gate_s = torch.sigmoid(sensory_sigma * (inputs.unsqueeze(-1) - sensory_mu))
    cond_s = sensory_w_pos * gate_s
    num_sensory = (cond_s * sensory_erev).sum(dim=1)
    den_sensory = cond_s.sum(dim=1)
    v = state
    for _ in range(ode_unfolds):
        gate_r = torch.sigmoid(sigma * (v.unsqueeze(-1) - mu))
        num = (gate_r * w_erev).sum(dim=1) + num_sensory
        den = (w_pos * gate_r).sum(dim=1) + den_sensory
        v = (cm_t * v + gleak_pos * vleak + num) / (cm_t + gleak_pos + den + epsilon)
    return v


@torch.jit.script
def _ltc_forward_loop_jit(
    x_seq: torch.Tensor,         # (B, T, D)
    state: torch.Tensor,         # (B, H)
    w_pos: torch.Tensor,
    w_erev: torch.Tensor,
    mu: torch.Tensor,
    sigma: torch.Tensor,
    sensory_mu: torch.Tensor,
    sensory_sigma: torch.Tensor,
    sensory_erev: torch.Tensor,
    sensory_w_pos: torch.Tensor,
    cm_t: torch.Tensor,
    gleak_pos: torch.Tensor,
    vleak: torch.Tensor,
    ode_unfolds: int,
    epsilon: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Outer loop over T time steps; returns (outputs (B, T, H), final state)."""
    B = x_seq.size(0)
    T = x_seq.size(1)
    H = state.size(1)
    outputs = torch.empty(B, T, H, device=x_seq.device, dtype=x_seq.dtype)
    for t in range(T):
        state = _ltc_ode_step_jit(
            x_seq[:, t, :], state, w_pos, w_erev, mu, sigma,
            sensory_mu, sensory_sigma, sensory_erev, sensory_w_pos,
            cm_t, gleak_pos, vleak, ode_unfolds, epsilon)
        outputs[:, t, :] = state
    return outputs, state


class TrueLiquidTimeConstant(nn.Module):
    """Liquid Time-Constant network layer (Hasani/Lechner LTC cell, ncps formulation).

    Per-synapse sigmoid-gated conductances with learned mu/sigma, per-synapse
    reversal potentials, leak reversal potential vleak, membrane capacitance
    cm and leak conductance gleak, a sensory synapse pathway from the inputs,
    and `ode_unfolds` implicit-Euler sub-steps per time step. No tanh on the
    state; softplus keeps w, cm, gleak and sensory_w positive.
    """

    def __init__(
        self,
        input_dim: int,
        hidden_dim: int = 64,
        dt: float = 1.0 / 30.0,
        ode_unfolds: int = 6,
        sparsity: float = 0.5,
        sensory_sparsity: float = 0.5,
        input_mapping: str = "affine",
        epsilon: float = 1e-8,
    ):
        super().__init__()
        self.input_dim = input_dim
        self.hidden_dim = hidden_dim
        self.dt = float(dt)
        self.ode_unfolds = int(max(1, ode_unfolds))
        self.sparsity = sparsity
        self.sensory_sparsity = sensory_sparsity
        self.input_mapping = input_mapping
        self.epsilon = epsilon

        H, D = hidden_dim, input_dim
        # The order of RNG draws below is part of the contract: a seed must
        # build the same tensors as the reference (ltc.py:149-172).
        self.w = nn.Parameter(torch.empty(H, H).uniform_(0.001, 1.0))
        self.mu = nn.Parameter(torch.empty(H, H).uniform_(0.3, 0.8))
        self.sigma = nn.Parameter(torch.empty(H, H).uniform_(3.0, 8.0))
        rec_mask, rec_erev = self._create_recurrent_wiring(H, sparsity)
        self.register_buffer("sparsity_mask", rec_mask)
        self.erev = nn.Parameter(rec_erev)

        self.sensory_w = nn.Parameter(torch.empty(D, H).uniform_(0.001, 1.0))
        self.sensory_mu = nn.Parameter(torch.empty(D, H).uniform_(0.3, 0.8))
        self.sensory_sigma = nn.Parameter(torch.empty(D, H).uniform_(3.0, 8.0))
        sens_mask, sens_erev = self._create_sensory_wiring(D, H, sensory_sparsity)
        self.register_buffer("sensory_sparsity_mask", sens_mask)
        self.sensory_erev = nn.Parameter(sens_erev)

        self.gleak = nn.Parameter(torch.empty(H).uniform_(0.001, 1.0))
        self.vleak = nn.Parameter(torch.empty(H).uniform_(-0.2, 0.2))
        self.cm = nn.Parameter(torch.empty(H).uniform_(0.4, 0.6))

        # Input mapping decides which of input_w / input_b are trainable (ltc.py:175-183).
        if input_mapping == "affine":
            self.input_w = nn.Parameter(torch.ones(D))
            self.input_b = nn.Parameter(torch.zeros(D))
        elif input_mapping == "linear":
            self.input_w = nn.Parameter(torch.ones(D))
            self.register_buffer("input_b", torch.zeros(D))
        else:
            self.register_buffer("input_w", torch.ones(D))
            self.register_buffer("input_b", torch.zeros(D))

        self.input_norm = nn.LayerNorm(D)
        # Eval-mode cache of the positivity transforms (ltc.py:188-190).
        self._cached_transforms: dict | None = None

    @staticmethod
    def _wiring(rows: int, hidden_dim: int, sparsity: float):
        """Bernoulli(sparsity) mask with every column non-empty, and +/-1 reversal signs."""
        if sparsity >= 1.0:
            mask = torch.ones(rows, hidden_dim)
        else:
            mask = (torch.rand(rows, hidden_dim) < sparsity).float()
            for col in range(hidden_dim):
                if not mask[:, col].any():
                    pick = torch.randint(0, rows, (1,))
                    mask[pick, col] = 1.0
        sign = torch.where(torch.rand(rows, hidden_dim) < 0.8,
                           torch.ones(rows, hidden_dim), -torch.ones(rows, hidden_dim))
        return mask, sign * mask

    @staticmethod
    def _create_recurrent_wiring(hidden_dim: int, sparsity: float):
        """Recurrent mask (H, H) and reversal potentials, ~80% excitatory (ltc.py:193-211)."""
        return TrueLiquidTimeConstant._wiring(hidden_dim, hidden_dim, sparsity)

    @staticmethod
    def _create_sensory_wiring(input_dim: int, hidden_dim: int, sparsity: float):
        """Sensory mask (D, H) and reversal potentials, ~80% excitatory (ltc.py:214-231)."""
        return TrueLiquidTimeConstant._wiring(input_dim, hidden_dim, sparsity)

    def _transforms(self):
        w_pos = F.softplus(self.w) * self.sparsity_mask
        w_erev = w_pos * self.erev
        cm_t = F.softplus(self.cm) / (self.dt / self.ode_unfolds)
        gleak_pos = F.softplus(self.gleak)
        sensory_w_pos = F.softplus(self.sensory_w) * self.sensory_sparsity_mask
        return w_pos, w_erev, cm_t, gleak_pos, sensory_w_pos

    def forward(
        self,
        x_seq: torch.Tensor,
        h0: tuple[torch.Tensor, torch.Tensor] | None = None,
    ) -> tuple[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]:
        """(B, T, D) inputs -> ((B, T, H) outputs, (h_final, h_final)).

        h0 is an (h, c) pair for LSTM API compatibility; only h is used.
        """
        B, T, D = x_seq.shape
        d = self.__dict__
        force_ts = d.get("_force_torchscript", False)
        on_hip = x_seq.is_cuda and x_seq.dtype == torch.float32 and not force_ts
        if on_hip and d["training"]:
            leaves = self._module_leaves(D)
            if leaves is not None:
                # Whole layer in two library calls: LayerNorm, affine and the
                # positivity transforms run inside the fused kernels. Without h0
                # the library starts from a zero state itself (state None).
                state = None if h0 is None else h0[0]
                if state is not None and state.dtype != x_seq.dtype:
                    state = state.to(x_seq.dtype)
                outputs, state = ltc_cuda.ltc_module_forward(
                    x_seq, state, leaves, d["dt"], d["ode_unfolds"], d["epsilon"],
                    d["_modules"]["input_norm"].__dict__["eps"])
                return outputs, (state, state)

        state = torch.zeros(B, self.hidden_dim, device=x_seq.device, dtype=x_seq.dtype)
        if h0 is not None:
            state = h0[0]
        x_seq = self.input_norm(x_seq)
        if state.dtype != x_seq.dtype:
            state = state.to(x_seq.dtype)
        x_seq = x_seq * self.input_w + self.input_b

        if not self.training and self._cached_transforms is not None:
            c = self._cached_transforms
            w_pos, w_erev, cm_t, gleak_pos, sensory_w_pos = (
                c["w_pos"], c["w_erev"], c["cm_t"], c["gleak_pos"], c["sensory_w_pos"])
        else:
            w_pos, w_erev, cm_t, gleak_pos, sensory_w_pos = self._transforms()
            if not self.training:
                self._cached_transforms = {
                    "w_pos": w_pos, "w_erev": w_erev, "cm_t": cm_t,
                    "gleak_pos": gleak_pos, "sensory_w_pos": sensory_w_pos,
                }

        if on_hip:
            ltc_cuda.require_kernels()
            outputs, state = ltc_cuda.ltc_cuda_forward(
                x_seq, state, w_pos, w_erev, self.mu, self.sigma,
                self.sensory_mu, self.sensory_sigma, self.sensory_erev, sensory_w_pos,
                cm_t, gleak_pos, self.vleak, self.ode_unfolds, self.epsilon)
        else:
            if not getattr(self, "_ts_fallback_warned", False):
                logger.info(
                    "LTC using the TorchScript loop: is_cuda=%s, dtype=%s, force_ts=%s",
                    x_seq.is_cuda, x_seq.dtype, force_ts)
                self._ts_fallback_warned = True
            outputs, state = _ltc_forward_loop_jit(
                x_seq, state, w_pos, w_erev, self.mu, self.sigma,
                self.sensory_mu, self.sensory_sigma, self.sensory_erev, sensory_w_pos,
                cm_t, gleak_pos, self.vleak, self.ode_unfolds, self.epsilon)
        return outputs, (state, state)

    def _module_path_ok(self, D: int) -> bool:
        """Whether the fused module path applies: standard LayerNorm, fp32 leaves, D in range."""
        return self._module_leaves(D) is not None

    def _module_leaves(self, D: int):
        """The 17 leaves of the fused module path in the library's order, or None
        when the path does not apply (a LayerNorm other than nn.LayerNorm over D
        with weight and bias, non-fp32 or host leaves, D out of range). Read
        straight from the registries: nn.Module attribute access costs a
        __getattr__ call per name on this per-step path."""
        d = self.__dict__
        P, Bf = d["_parameters"], d["_buffers"]
        norm = d["_modules"].get("input_norm")
        w = P.get("w")
        if (D > ltc_cuda.MODULE_MAX_D or not isinstance(norm, nn.LayerNorm) or w is None
                or w.dtype != torch.float32 or not w.is_cuda):
            return None
        nd = norm.__dict__
        NP = nd["_parameters"]
        lw, lb = NP.get("weight"), NP.get("bias")
        if lw is None or lb is None or tuple(nd["normalized_shape"]) != (D,):
            return None
        return [w, P["erev"], Bf["sparsity_mask"], P["mu"], P["sigma"],
                P["sensory_w"], P["sensory_erev"], Bf["sensory_sparsity_mask"],
                P["sensory_mu"], P["sensory_sigma"], P["gleak"], P["vleak"], P["cm"],
                P["input_w"] if "input_w" in P else Bf["input_w"],
                P["input_b"] if "input_b" in P else Bf["input_b"], lw, lb]

    def zero_grad(self, set_to_none: bool = True) -> None:
        """nn.Module.zero_grad over the layer's own parameters and its LayerNorm's,
        read straight from their registries: the generic walk over
        named_parameters costs more host time than the rest of a small layer's
        step. Any other module structure takes nn.Module's own walk."""
        d = self.__dict__
        mods = d["_modules"]
        norm = mods.get("input_norm")
        if (len(mods) != 1 or type(norm) is not nn.LayerNorm or norm._modules
                or d.get("_is_replica", False)):
            return super().zero_grad(set_to_none)
        for reg in (d["_parameters"], norm.__dict__["_parameters"]):
            for p in reg.values():
                if p is None or p.grad is None:
                    continue
                if set_to_none:
                    p.grad = None
                else:
                    if p.grad.grad_fn is not None:
                        p.grad.detach_()
                    else:
                        p.grad.requires_grad_(False)
                    p.grad.zero_()

    def train(self, mode: bool = True):
        """Switching to train mode drops the eval-mode transform cache (ltc.py:328-332)."""
        if mode:
            self._cached_transforms = None
        return super().train(mode)

    @property
    def W_rec(self) -> nn.Parameter:
        """Compatibility alias of the recurrent weight parameter (ltc.py:336-339)."""
        return self.w

    def fused_euler_step(self, *args, **kwargs):
        """Removed entry point kept for attribute checks (ltc.py:341-345)."""
        raise NotImplementedError(
            "fused_euler_step is removed. Use _ode_solver(inputs, state) instead."
        )


TemporalLTC = TrueLiquidTimeConstant


def _on_hip(*tensors) -> bool:
    """Whether the fused operators serve these: HIP tensors go to the library, and a
    missing library is an error there; CPU tensors take the plain forms below."""
    return all(t is None or t.is_cuda for t in tensors)


def _gated_scan_plain(x, gate, state, cu_seqlens=None):
    """ltc_cuda.ltc_gated_scan's "blend" form in plain torch, step by step."""
    if cu_seqlens is None:
        a, u = torch.sigmoid(gate), torch.sigmoid(-gate) * x
        h, outs = state, []
        for t in range(x.shape[1]):
            h = a[:, t] * h + u[:, t]
            outs.append(h)
        return (torch.stack(outs, 1) if outs else torch.zeros_like(x)), h
    cu = cu_seqlens.tolist()
    out, finals = [x.new_zeros(cu[0], x.shape[1])], []
    for s in range(len(cu) - 1):
        o, h = _gated_scan_plain(x[None, cu[s]:cu[s + 1]], gate[None, cu[s]:cu[s + 1]],
                                 state[s:s + 1])
        out.append(o[0])
        finals.append(h)
    out.append(x.new_zeros(x.shape[0] - cu[-1], x.shape[1]))
    return torch.cat(out), (torch.cat(finals) if finals else state)


class _ScaleColumns(torch.autograd.Function):
    """w (D, H) times s (H,). The gradient of s is summed by halves. torch's reduction
    over many rows takes several workgroups, whose counters a memset node clears in a
    captured graph, and on ROCm 7.2 such graphs give other sums from the second replay
    on (torch 2.10: the gradient of a Linear(32, 700)'s bias over 600 rows, while one
    reduction alone in a graph is right)."""

    @staticmethod
    def forward(ctx, w, s):
        ctx.save_for_backward(w, s)
        return w * s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        w, s = ctx.saved_tensors
        t = g * w
        t = F.pad(t, (0, 0, 0, (1 << (t.shape[0] - 1).bit_length()) - t.shape[0]))
        while t.shape[0] > 1:
            half = t.shape[0] // 2
            t = t[:half] + t[half:]
        return g * s, t[0]


class LinearTimeConstant(nn.Module):
    """LTC layer without recurrent synapses: sensory synapses, leak and capacitance only.

    Its implicit-Euler step v' = (cm v + gleak vleak + num) / (cm + gleak + den +
    epsilon) is a gated linear recurrence, since num and den come from the inputs
    alone: with G = gleak + den + epsilon, a = cm / (cm + G) = sigmoid(log cm - log G)
    and v' = a v + (1 - a) (gleak vleak + num) / G. So a whole sequence is one sensory
    pass over all steps and one ltc_cuda.ltc_gated_scan, parallel in time, where
    TrueLiquidTimeConstant advances step by step. Same parameter names, constructor
    arguments and calling convention as that layer, of which it is the case of one
    unfold and an empty recurrent mask.

    float32, as that layer. forward also takes packed sequences: x_seq (tokens, D)
    with cu_seqlens (int32, sequences + 1). step() advances streams by one token for
    serving, their states updated in place, in rows of a pool if slots are given.

    The gate goes by a logarithm here and an exponential in the scan, each to a few
    roundings, since the scan takes pre-activations.
    """

    def __init__(
        self,
        input_dim: int,
        hidden_dim: int = 64,
        dt: float = 1.0 / 30.0,
        sensory_sparsity: float = 0.5,
        input_mapping: str = "affine",
        epsilon: float = 1e-8,
    ):
        super().__init__()
        self.input_dim = input_dim
        self.hidden_dim = hidden_dim
        self.dt = float(dt)
        self.sensory_sparsity = sensory_sparsity
        self.input_mapping = input_mapping
        self.epsilon = epsilon
        H, D = hidden_dim, input_dim
        self.sensory_w = nn.Parameter(torch.empty(D, H).uniform_(0.001, 1.0))
        self.sensory_mu = nn.Parameter(torch.empty(D, H).uniform_(0.3, 0.8))
        self.sensory_sigma = nn.Parameter(torch.empty(D, H).uniform_(3.0, 8.0))
        mask, erev = TrueLiquidTimeConstant._create_sensory_wiring(D, H, sensory_sparsity)
        self.register_buffer("sensory_sparsity_mask", mask)
        self.sensory_erev = nn.Parameter(erev)
        self.gleak = nn.Parameter(torch.empty(H).uniform_(0.001, 1.0))
        self.vleak = nn.Parameter(torch.empty(H).uniform_(-0.2, 0.2))
        self.cm = nn.Parameter(torch.empty(H).uniform_(0.4, 0.6))
        w, b = torch.ones(D), torch.zeros(D)
        if input_mapping in ("affine", "linear"):
            self.input_w = nn.Parameter(w)
        else:
            self.register_buffer("input_w", w)
        if input_mapping == "affine":
            self.input_b = nn.Parameter(b)
        else:
            self.register_buffer("input_b", b)
        self.input_norm = nn.LayerNorm(D)

    def _drive(self, x):
        """Gate and drive of every row: (..., D) -> two (..., H).

        The leak is a synapse from a constant input (sigma 0, so its gate is 1/2), the
        capacitance scales every conductance, and the input map is part of the
        LayerNorm's: every parameter's gradient over the rows is then formed by the
        sensory kernels or the LayerNorm, in the same order each time.
        """
        norm = self.input_norm
        rows = F.layer_norm(x, (self.input_dim,), norm.weight * self.input_w,
                            norm.bias * self.input_w + self.input_b,
                            norm.eps).reshape(-1, self.input_dim)
        gleak = F.softplus(self.gleak)
        leak = gleak + self.epsilon
        zero = torch.zeros_like(leak)
        w_pos = torch.cat([F.softplus(self.sensory_w) * self.sensory_sparsity_mask,
                           (2.0 * leak)[None]])
        w_pos = _ScaleColumns.apply(w_pos, self.dt / F.softplus(self.cm))
        erev = torch.cat([self.sensory_erev, (gleak * self.vleak / leak)[None]])
        mu = torch.cat([self.sensory_mu, zero[None]])
        sigma = torch.cat([self.sensory_sigma, zero[None]])
        rows = F.pad(rows, (0, 1))
        if _on_hip(rows):
            num, den = ltc_cuda.ltc_sensory_sums(rows, sigma, mu, w_pos, erev)
        else:
            cond = w_pos * torch.sigmoid(sigma * (rows.unsqueeze(-1) - mu))
            num, den = (cond * erev).sum(1), cond.sum(1)
        # a = cm / (cm + G) = 1 / (1 + den), the conductances being in units of cm
        shape = (*x.shape[:-1], self.hidden_dim)
        return -torch.log(den).view(shape), (num / den).view(shape)

    def forward(self, x_seq, h0=None, cu_seqlens=None):
        """(B, T, D), or packed (tokens, D) with cu_seqlens -> (outputs, (h, h)).

        h0 is an (h, c) pair as TrueLiquidTimeConstant takes it; only h is used.
        """
        state = None if h0 is None else h0[0]
        gate, drive = self._drive(x_seq)
        if _on_hip(x_seq):
            out, h = ltc_cuda.ltc_gated_scan(drive, gate, state, cu_seqlens)
        else:
            if state is None:
                n = x_seq.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
                state = drive.new_zeros(n, self.hidden_dim)
            out, h = _gated_scan_plain(drive, gate, state, cu_seqlens)
        return out, (h, h)

    @torch.no_grad()
    def step(self, x, state, slots=None):
        """One token of each stream: x (B, D) -> (B, H); `state` (B, H), or a pool
        whose rows slots (B,) int32 name (negative: padding), is updated in place."""
        gate, drive = self._drive(x)
        if _on_hip(x, state):
            return ltc_cuda.ltc_gated_scan_step(drive, gate, state, slots)
        out = torch.zeros_like(drive)
        for b in range(x.shape[0]):
            s = b if slots is None else int(slots[b])
            if s >= 0:
                state[s] = torch.lerp(drive[b], state[s], torch.sigmoid(gate[b]))
                out[b] = state[s]
        return out


class TokenEmbedding(nn.Module):
    """Rows of a table for tokens, times a scale: forward(ids (...)) -> (..., dim).

    A negative id is a token that is not there: zeros, and no gradient. The table's
    gradient is dense and the same bits in every run (ltc_cuda.ltc_embed). CPU tensors take
    plain torch, which raises for an id past the vocabulary where the kernels give NaN.
    """

    def __init__(self, vocab: int, dim: int, scale: float = 1.0, dtype=None):
        super().__init__()
        self.scale = float(scale)
        self.weight = nn.Parameter(torch.randn(vocab, dim, dtype=dtype) * dim ** -0.5)

    def forward(self, ids):
        if _on_hip(self.weight, ids):
            return ltc_cuda.ltc_embed(self.weight, ids, self.scale)
        there = (ids >= 0).unsqueeze(-1)
        rows = F.embedding(ids.clamp(min=0).long(), self.weight) * self.scale
        return torch.where(there, rows, torch.zeros_like(rows))


def _causal_conv_plain(x, weight, bias, state, cu_seqlens=None):
    """ltc_cuda.ltc_causal_conv with "silu" in plain torch."""
    K = weight.shape[1]
    if cu_seqlens is None:
        line = torch.cat([state, x], 1)
        y = sum(line[:, k:k + x.shape[1]] * weight[:, k] for k in range(K)) + bias
        return F.silu(y), line[:, x.shape[1]:]
    cu = cu_seqlens.tolist()
    outs, tails = [x.new_zeros(cu[0], x.shape[1])], []
    for s in range(len(cu) - 1):
        o, t = _causal_conv_plain(x[None, cu[s]:cu[s + 1]], weight, bias, state[s:s + 1])
        outs.append(o[0])
        tails.append(t)
    outs.append(x.new_zeros(x.shape[0] - cu[-1], x.shape[1]))
    return torch.cat(outs), (torch.cat(tails) if tails else state)


def _selective_scan_plain(x, delta, A, B, C, D, z, delta_bias, state, cu_seqlens=None):
    """ltc_cuda.ltc_selective_scan with a softplus of the step sizes in plain torch."""
    if cu_seqlens is None:
        s = F.softplus(delta.float() + delta_bias)
        h, outs = state, []
        for t in range(x.shape[1]):
            u = (s[:, t] * x[:, t].float()).unsqueeze(-1) * B[:, t, None].float()
            h = torch.exp(s[:, t, :, None] * A) * h + u
            y = (h * C[:, t, None].float()).sum(-1) + D * x[:, t].float()
            outs.append((y * F.silu(z[:, t].float())).to(x.dtype))
        return (torch.stack(outs, 1) if outs else torch.zeros_like(x)), h
    cu = cu_seqlens.tolist()
    outs, finals = [x.new_zeros(cu[0], x.shape[1])], []
    for s in range(len(cu) - 1):
        part = [v[None, cu[s]:cu[s + 1]] for v in (x, delta, B, C, z)]
        o, h = _selective_scan_plain(part[0], part[1], A, part[2], part[3], D, part[4], delta_bias,
                                     state[s:s + 1])
        outs.append(o[0])
        finals.append(h)
    outs.append(x.new_zeros(x.shape[0] - cu[-1], x.shape[1]))
    return torch.cat(outs), (torch.cat(finals) if finals else state)


class SelectiveTimeConstant(nn.Module):
    """Layer of states whose time constants the input selects: a projection to the channels
    and their gates, a short causal convolution, a selective state space scan, and a
    projection back.

    Each channel h has `states` states v with v' = exp(s_t A) v + s_t B_t x_t, where the step
    sizes s_t (softplus of a projection of rank `rank`), the drives B_t and the readouts C_t
    all come from the input; LinearTimeConstant has one state a channel, whose decay comes
    from its synapses.

    forward(x (B, T, dim)) -> (out, state), or packed x (tokens, dim) with cu_seqlens as
    ltc_cuda.ltc_gated_scan takes them. A state is a pair: the convolution's last inputs
    (rows, taps-1, hidden) and the scan's states (rows, hidden, states) in float32;
    new_state(rows) makes a zero one. step(x (B, dim), state, slots) serves streams token by
    token, their state updated in place, in rows of a pool if slots are given. The
    projections have no bias: torch forms its gradient with a reduction that a captured graph
    replays wrongly (_ScaleColumns).
    """

    def __init__(self, dim: int, hidden: int | None = None, states: int = 16, taps: int = 4,
                 rank: int | None = None, dt_min: float = 1e-3, dt_max: float = 0.1, dtype=None):
        super().__init__()
        hidden = 2 * dim if hidden is None else hidden
        rank = max(1, dim // 16) if rank is None else rank
        self.dim, self.hidden, self.states, self.taps, self.rank = dim, hidden, states, taps, rank
        self.in_proj = nn.Linear(dim, 2 * hidden, bias=False, dtype=dtype)
        self.x_proj = nn.Linear(hidden, rank + 2 * states, bias=False, dtype=dtype)
        self.dt_proj = nn.Linear(rank, hidden, bias=False, dtype=dtype)
        self.out_proj = nn.Linear(hidden, dim, bias=False, dtype=dtype)
        self.conv_weight = nn.Parameter((torch.rand(hidden, taps) * 2 - 1) * taps ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(hidden))
        # decays of 1 to `states` of a step, steps spread over their range in logarithm
        self.A_log = nn.Parameter(torch.log(torch.arange(1, states + 1).float()).repeat(hidden, 1))
        self.D = nn.Parameter(torch.ones(hidden))
        lo, hi = torch.tensor(dt_min).log(), torch.tensor(dt_max).log()
        dt = torch.exp(lo + (hi - lo) * torch.rand(hidden))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))

    def new_state(self, rows: int):
        w = self.in_proj.weight
        return (w.new_zeros(rows, self.taps - 1, self.hidden),
                torch.zeros(rows, self.hidden, self.states, device=w.device))

    def _rates(self):
        """What the scan takes in float32, whatever the module's type."""
        return -torch.exp(self.A_log.float()), self.D.float(), self.dt_bias.float()

    def _selected(self, u):
        """Step sizes, drives and readouts of the convolved input."""
        r, n = self.rank, self.states
        low = self.x_proj(u)
        return self.dt_proj(low[..., :r]), low[..., r:r + n], low[..., r + n:]

    def forward(self, x, state=None, cu_seqlens=None):
        x = x.to(self.in_proj.weight.dtype)
        both = self.in_proj(x)
        u, z = both[..., :self.hidden], both[..., self.hidden:]
        A, D, dt_bias = self._rates()
        tail, h = (None, None) if state is None else state
        if _on_hip(x, tail, h, cu_seqlens):
            u, tail = ltc_cuda.ltc_causal_conv(u, self.conv_weight, self.conv_bias, tail, cu_seqlens, "silu")
            delta, B, C = self._selected(u)
            y, h = ltc_cuda.ltc_selective_scan(u, delta, A, B, C, D, z, dt_bias, h, cu_seqlens, True)
        else:
            if state is None:
                tail, h = self.new_state(x.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1)
            u, tail = _causal_conv_plain(u, self.conv_weight, self.conv_bias, tail, cu_seqlens)
            u = u.to(x.dtype)
            delta, B, C = self._selected(u)
            y, h = _selective_scan_plain(u, delta, A, B, C, D, z, dt_bias, h, cu_seqlens)
        return self.out_proj(y), (tail, h)

    @torch.no_grad()
    def step(self, x, state, slots=None):
        """One token of each stream: x (B, dim) -> (B, dim); `state` is updated in place.
        A negative slot is padding: zeros."""
        x = x.to(self.in_proj.weight.dtype)
        both = self.in_proj(x)
        u, z = both[..., :self.hidden], both[..., self.hidden:]
        A, D, dt_bias = self._rates()
        tail, h = state
        if _on_hip(x, tail, h, slots):
            u = ltc_cuda.ltc_causal_conv_step(u, self.conv_weight, tail, self.conv_bias, slots, "silu")
            delta, B, C = self._selected(u)
            y = ltc_cuda.ltc_selective_scan_step(u, delta, A, B, C, h, D, z, dt_bias, slots, True)
            return self.out_proj(y)
        out = torch.zeros_like(x)
        for b in range(x.shape[0]):
            s = b if slots is None else int(slots[b])
            if s < 0:
                continue
            ub, tail[s:s + 1] = _causal_conv_plain(u[b, None, None], self.conv_weight, self.conv_bias, tail[s:s + 1])
            ub = ub.to(x.dtype)
            delta, B, C = self._selected(ub)
            y, h[s:s + 1] = _selective_scan_plain(ub, delta, A, B, C, D, z[b, None, None], dt_bias, h[s:s + 1])
            out[b] = self.out_proj(y)[0, 0]
        return out


class TokenReadout(nn.Module):
    """Linear readout of a layer's states to the logits of a vocabulary, and what is
    asked of them: scores of given tokens, and a teacher's distribution to learn.

    forward(h) -> logits; log_probs(h, ids) -> ltc_cuda.ltc_token_logprobs of them;
    distill(h, teacher_logits, teacher_ids) -> ltc_cuda.ltc_top_distill's loss of each
    row; adjusted(h, context, ...) -> the logits as ltc_cuda.ltc_adjust_logits leaves them
    for the choice of the next token. The logits are in the readout's own type (float32, bfloat16 or float16), what
    is made of them in float32. There is no bias: torch forms its gradient with a
    reduction that a captured graph replays wrongly (_ScaleColumns). CPU tensors take
    plain torch, which raises for an id past the vocabulary where the kernels give NaN.
    """

    def __init__(self, hidden_dim: int, vocab: int, dtype=None):
        super().__init__()
        self.proj = nn.Linear(hidden_dim, vocab, bias=False, dtype=dtype)

    def forward(self, h):
        return self.proj(h.to(self.proj.weight.dtype))

    def log_probs(self, h, ids, top: int = 0, temperature: float = 1.0):
        """(log probability, entropy[, top log probabilities, top ids]) of each row."""
        logits = self(h)
        if _on_hip(logits):
            return ltc_cuda.ltc_token_logprobs(logits, ids, top=top, temperature=temperature)
        lq = torch.log_softmax(logits.float() / temperature, -1)
        q = lq.exp()
        ent = -torch.where(q > 0, q * lq, torch.zeros_like(q)).sum(-1)
        lp = lq.gather(-1, ids.clamp(min=0).long().unsqueeze(-1)).squeeze(-1)
        zero = torch.zeros_like(ent)
        res = (torch.where(ids >= 0, lp, zero), torch.where(ids >= 0, ent, zero))
        if top:
            order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :top]
            res += (lq.gather(-1, order).detach(), order)
        return res

    def distill(self, h, teacher_logits, teacher_ids, temperature: float = 1.0):
        """Distillation loss of each row against the teacher's best logits."""
        logits = self(h)
        if _on_hip(logits):
            return ltc_cuda.ltc_top_distill(logits, teacher_logits, teacher_ids,
                                            temperature=temperature)
        lq = torch.log_softmax(logits.float() / temperature, -1)
        t = teacher_logits.float() / temperature
        t = t.masked_fill(teacher_ids < 0, -float("inf"))
        some = (t > -float("inf")).any(-1, keepdim=True)
        lp = torch.log_softmax(torch.where(some, t, torch.zeros_like(t)), -1)
        p = torch.where(some & (t > -float("inf")), lp.exp(), torch.zeros_like(lp))
        diff = lp - lq.gather(-1, teacher_ids.clamp(min=0).long())
        return temperature ** 2 * torch.where(p > 0, p * diff, torch.zeros_like(p)).sum(-1)

    @torch.no_grad()
    def adjusted(self, h, context=None, prompt_lens=None, repetition=1.0, frequency=0.0,
                 presence=0.0, bias_ids=None, bias=None, mask=None):
        """Logits with penalties for the context's tokens, biases and a grammar's mask."""
        logits = self(h)
        if _on_hip(logits):
            return ltc_cuda.ltc_adjust_logits(logits, context, prompt_lens, repetition, frequency,
                                              presence, bias_ids, bias, mask)
        lead, V = logits.shape[:-1], logits.shape[-1]
        v = logits.float().reshape(-1, V)

        def rows(t):
            t = t if t.dim() == len(lead) + 1 else t.expand(*lead, t.shape[-1])
            return t.reshape(v.shape[0], -1)

        def column(p):
            return p.reshape(-1, 1) if isinstance(p, torch.Tensor) else p

        if context is not None:
            ids = rows(context)
            there = (ids >= 0) & (ids < V)
            start = 0 if prompt_lens is None else prompt_lens.reshape(-1, 1)
            later = there & (torch.arange(ids.shape[1]) >= start)
            at = ids.clamp(0, V - 1).long()
            seen = torch.zeros_like(v).scatter_add_(1, at, there.float()) > 0
            count = torch.zeros_like(v).scatter_add_(1, at, later.float())
            rep = column(repetition)
            v = torch.where(seen, torch.where(v > 0, v / rep, v * rep), v)
            v = torch.where(count > 0, v - column(frequency) * count - column(presence), v)
        if bias_ids is not None:
            ids, b = rows(bias_ids), rows(bias)
            there = (ids >= 0) & (ids < V)
            v = v.scatter_add(1, ids.clamp(0, V - 1).long(), torch.where(there, b, torch.zeros_like(b)))
        if mask is not None:
            t = torch.arange(V)
            v = v.masked_fill((rows(mask)[:, t // 32] >> (t % 32)) & 1 == 0, -float("inf"))
        return v.to(logits.dtype).view(*lead, V)
