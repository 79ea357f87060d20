"""Neuron, surrogate and dropout modules with SpikingJelly's public behaviour
(``activation_based.neuron.LIFNode``, ``surrogate.ATan``, ``layer.Dropout``,
``base.MemoryModule``), which the reference builds its layers from
(src/delrec/delay_layers.py:21-31, networks.py:84-96).

The delay layers only read the LIF constants from ``neuron_module``; the multi-step
``LIFNode.forward`` (used between projections in the model zoo) runs the CUDA LIF kernel.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import functional as Fn
from .block_norm import GATES, block_join, block_norm
from .gated import gated_scan, gated_step
from .selective import selective_scan, selective_step
from .short_conv import ACTS, short_conv, short_conv_step


class MemoryModule(torch.nn.Module):
    """Module with resettable state registered through ``register_memory``."""

    def __init__(self):
        super().__init__()
        self._memories = {}
        self._memories_rv = {}

    def register_memory(self, name, value):
        self._memories[name] = value
        self._memories_rv[name] = value

    def reset(self):
        for k in self._memories:
            self._memories[k] = self._memories_rv[k]

    def __getattr__(self, name):
        mem = self.__dict__.get("_memories")
        if mem is not None and name in mem:
            return mem[name]
        return super().__getattr__(name)

    def __setattr__(self, name, value):
        mem = self.__dict__.get("_memories")
        if mem is not None and name in mem:
            mem[name] = value
        else:
            super().__setattr__(name, value)


class _ATanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, alpha):
        ctx.save_for_backward(x)
        ctx.alpha = alpha
        return (x >= 0).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        a = ctx.alpha
        return a / 2 / (1 + (math.pi / 2 * a * x).pow(2)) * g, None


class ATan(torch.nn.Module):
    """Heaviside spike with the arctangent surrogate gradient."""

    def __init__(self, alpha: float = 2.0, spiking: bool = True):
        super().__init__()
        self.alpha = alpha
        self.spiking = spiking

    def forward(self, x):
        return _ATanFn.apply(x, self.alpha)


class LIFNode(MemoryModule):
    """Leaky integrate-and-fire neuron (tau, v_threshold, v_reset (None = soft reset),
    surrogate_function, detach_reset).  Multi-step mode runs the CUDA kernel; only
    ``decay_input=False`` is supported (the reference's fused kernels assume it too)."""

    def __init__(self, tau: float = 2.0, decay_input: bool = True, v_threshold: float = 1.0,
                 v_reset=0.0, surrogate_function=None, detach_reset: bool = False,
                 step_mode: str = "s", backend: str = "torch", store_v_seq: bool = False):
        super().__init__()
        self.tau = tau
        self.decay_input = decay_input
        self.v_threshold = v_threshold
        self.v_reset = v_reset
        self.surrogate_function = surrogate_function if surrogate_function is not None else ATan()
        self.detach_reset = detach_reset
        self.step_mode = step_mode
        self.backend = backend
        self.store_v_seq = store_v_seq
        self.register_memory("v", 0.0 if v_reset is None else v_reset)

    def _lif_args(self):
        surr = self.surrogate_function
        from .utils import Triangle
        if "ATan" in type(surr).__name__:
            sid, alpha = 1, float(getattr(surr, "alpha", 2.0))
        else:
            sid, alpha = 0, 2.0
        gamma = 1.0
        if surr is not Triangle.apply and hasattr(surr, "gamma"):
            gamma = float(surr.gamma)
        return (self.tau, self.v_threshold, self.v_reset, self.detach_reset, sid, gamma, alpha)

    def forward(self, x):
        if self.step_mode != "m":
            raise NotImplementedError("delrec_b200 LIFNode runs in multi-step mode ('m') only")
        if self.decay_input:
            raise NotImplementedError("decay_input=True is not supported by the CUDA kernels")
        return Fn.LIFMultiStep.apply(x, self._lif_args())

    def extra_repr(self):
        return (f"tau={self.tau}, v_threshold={self.v_threshold}, v_reset={self.v_reset}, "
                f"detach_reset={self.detach_reset}, step_mode={self.step_mode}")


class Dropout(MemoryModule):
    """Dropout whose mask is drawn once (on the first call after ``reset``) and reused,
    so a recurrent layer sees the same mask at every time step."""

    def __init__(self, p: float = 0.5, step_mode: str = "s"):
        super().__init__()
        self.p = p
        self.step_mode = step_mode
        self.register_memory("mask", None)

    def create_mask(self, x):
        self.mask = F.dropout(torch.ones_like(x), self.p, training=True)

    def forward(self, x):
        if not self.training or self.p <= 0:
            return x
        if self.step_mode == "m":
            if self.mask is None:
                self.create_mask(x[0])
            return x * self.mask
        if self.mask is None:
            self.create_mask(x)
        return x * self.mask

    def extra_repr(self):
        return f"p={self.p}, step_mode={self.step_mode}"


class BatchNorm1d(torch.nn.BatchNorm1d):
    """Multi-step batch norm over (T, B, N, 1) inputs flattened on (T*B)."""

    def __init__(self, num_features, step_mode="m", **kw):
        super().__init__(num_features, **kw)
        self.step_mode = step_mode

    def forward(self, x):
        if self.step_mode == "m" and x.dim() >= 3:
            shp = x.shape
            y = super().forward(x.flatten(0, 1))
            return y.view(shp)
        return super().forward(x)


# States of streaming modules.  Eagerly each call makes a new one, and who keeps the state before can go back to
# it.  A call captured in a graph moves the state that there is on in place, so that every replay takes it further.


def _captured(m):
    """Is a call of module ``m`` captured that moves a state on?  The state then lives as long as the module does,
    also after ``reset``: replays write to it."""
    if m.v is None or not torch.cuda.is_current_stream_capturing():
        return False
    held = m.__dict__.setdefault("_captured_states", [])
    if not any(v is m.v for v in held):
        held.append(m.v)
    return True


def _kept(m):
    """The state that a multi-step call of module ``m`` begins from (a copy where it will be written over: a backward
    pass may want it)."""
    if not m.keep_state:
        return None
    return m.v.clone() if _captured(m) else m.v


def _keep(m, v):
    """``v`` is the state behind a multi-step call."""
    if m.keep_state:
        if _captured(m):
            m.v.copy_(v.detach())
        else:
            m.v = v.detach()


class GatedIntegrator(MemoryModule):
    """A leaky integrator with a learned, input-dependent decay (``gated.gated_scan``), in
    place of ``LIFNode`` where no spikes are wanted: forward(z, f) with gate logits f.

    Multi-step mode: z (T,B,N), f (T,B,G) -> h (T,B,N) from a zero state, or from the state
    of the call before with ``keep_state=True``.  Single-step mode ('s'): z (B,N), f (B,G) ->
    h (B,N), the state moving on from call to call until ``reset`` (``utils.reset_states``);
    no gradient passes.  ``v`` is the state (B,N) in float32.  A call captured in a CUDA graph
    moves the ``v`` that there is on in place, replay after replay (``v.zero_()`` starts it
    again); without one it begins from zeros each time."""

    def __init__(self, decay_input: bool = True, step_mode: str = "m", keep_state: bool = False,
                 checkpoint8: bool = False):
        super().__init__()
        if step_mode not in ("m", "s"):
            raise ValueError(f"step_mode must be 'm' or 's', got {step_mode!r}")
        self.decay_input = decay_input
        self.step_mode = step_mode
        self.keep_state = keep_state
        self.checkpoint8 = checkpoint8
        self.register_memory("v", None)

    def forward(self, z, f, lengths=None, resets=None):
        if self.step_mode == "s":
            if lengths is not None or resets is not None:
                raise RuntimeError("delrec_b200: lengths and resets are for the multi-step mode")
            h, self.v = gated_step(z, f, self.v, decay_input=self.decay_input, out=self.v if _captured(self) else None)
            return h
        h, v = gated_scan(z, f, _kept(self), lengths=lengths, resets=resets,
                          decay_input=self.decay_input, checkpoint8=self.checkpoint8)
        _keep(self, v)
        return h

    def extra_repr(self):
        return f"decay_input={self.decay_input}, step_mode={self.step_mode}, checkpoint8={self.checkpoint8}"


class ShortConv(MemoryModule):
    """A short causal convolution over time, one filter per channel (``short_conv.short_conv``),
    as it stands in front of ``GatedIntegrator`` or ``SelectiveIntegrator``.

    Multi-step mode: x (T,B,N) -> y (T,B,N) from zeros, or from the window of the call before with
    ``keep_state=True``.  Single-step mode ('s'): x (B,N) -> y (B,N), the window moving on from call
    to call until ``reset`` (``utils.reset_states``); no gradient passes.  ``v`` is the window
    (K-1,B,N) in x's type, in a CUDA graph as in ``GatedIntegrator``."""

    def __init__(self, num_features, kernel_size: int = 4, act: str = "silu", bias: bool = True, step_mode: str = "m",
                 keep_state: bool = False):
        super().__init__()
        if step_mode not in ("m", "s"):
            raise ValueError(f"step_mode must be 'm' or 's', got {step_mode!r}")
        if act not in ACTS:
            raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
        self.act, self.step_mode, self.keep_state = act, step_mode, keep_state
        bound = kernel_size ** -0.5
        self.weight = torch.nn.Parameter(torch.empty(num_features, kernel_size).uniform_(-bound, bound))
        if bias:
            self.bias = torch.nn.Parameter(torch.empty(num_features).uniform_(-bound, bound))
        else:
            self.register_parameter("bias", None)
        self.register_memory("v", None)

    def forward(self, x, lengths=None, resets=None):
        if self.step_mode == "s":
            if lengths is not None or resets is not None:
                raise RuntimeError("delrec_b200: lengths and resets are for the multi-step mode")
            y, self.v = short_conv_step(x, self.weight, self.bias, self.v, act=self.act, out=self.v if _captured(self) else None)
            return y
        y, v = short_conv(x, self.weight, self.bias, _kept(self), act=self.act, lengths=lengths, resets=resets)
        _keep(self, v)
        return y

    def extra_repr(self):
        n, k = self.weight.shape
        return f"{n}, kernel_size={k}, act={self.act}, step_mode={self.step_mode}"


class SelectiveIntegrator(MemoryModule):
    """A recurrence of S states per channel whose step size, input and output weights depend on the
    input (``selective.selective_scan``), where ``GatedIntegrator`` has one state and its gate.

    forward(x, dt, B, C, gate=None): multi-step mode (T,B,N) .. -> y (T,B,N) from a zero state, or
    from the state of the call before with ``keep_state=True``; single-step mode ('s') (B,N) .. ->
    y (B,N), the state moving on from call to call until ``reset``, in a CUDA graph as in
    ``GatedIntegrator``; no gradient passes.  Learned: the
    decay A = -exp(A_log) (N,S), the skip D (N) and the bias of dt (N), whose step sizes start
    between ``dt_min`` and ``dt_max``.  ``v`` is the state (B,N,S) in float32."""

    def __init__(self, num_features, num_states: int = 16, dt_min: float = 1e-3, dt_max: float = 0.1,
                 step_mode: str = "m", keep_state: bool = False):
        super().__init__()
        if step_mode not in ("m", "s"):
            raise ValueError(f"step_mode must be 'm' or 's', got {step_mode!r}")
        self.step_mode, self.keep_state = step_mode, keep_state
        rates = torch.arange(1, num_states + 1, dtype=torch.float32)
        self.A_log = torch.nn.Parameter(torch.log(rates).repeat(num_features, 1))
        self.D = torch.nn.Parameter(torch.ones(num_features))
        step = torch.exp(torch.empty(num_features).uniform_(math.log(dt_min), math.log(dt_max)))
        self.dt_bias = torch.nn.Parameter(step + torch.log(-torch.expm1(-step)))   # softplus of it is the step
        self.register_memory("v", None)

    def forward(self, x, dt, B, C, gate=None, lengths=None, resets=None):
        A = -torch.exp(self.A_log)
        if self.step_mode == "s":
            if lengths is not None or resets is not None:
                raise RuntimeError("delrec_b200: lengths and resets are for the multi-step mode")
            y, self.v = selective_step(x, dt, A, B, C, self.v, D=self.D, gate=gate, dt_bias=self.dt_bias,
                                       out=self.v if _captured(self) else None)
            return y
        y, v = selective_scan(x, dt, A, B, C, _kept(self), D=self.D, gate=gate, dt_bias=self.dt_bias, lengths=lengths,
                              resets=resets)
        _keep(self, v)
        return y

    def extra_repr(self):
        n, k = self.A_log.shape
        return f"{n}, num_states={k}, step_mode={self.step_mode}"


class BlockNorm(torch.nn.Module):
    """RMS norm per position before the first block (``block_norm.block_norm``)."""

    def __init__(self, num_features, eps: float = 1e-5):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(num_features))

    def forward(self, x, lengths=None):
        return block_norm(x, self.weight, eps=self.eps, lengths=lengths)


class BlockJoin(torch.nn.Module):
    """After a block: norm, gate, residual scale and sum, and the next block's norm
    (``block_norm.block_join``).  forward(x, y, gate=None) -> (x', n), or x' alone with
    ``next_norm=False`` (after the last block)."""

    def __init__(self, num_features, gate_act: str = "sigmoid", scale_init: float = 1.0, next_norm: bool = True,
                 eps: float = 1e-5):
        super().__init__()
        if gate_act not in GATES:
            raise ValueError(f"gate_act must be one of {sorted(GATES)}, got {gate_act!r}")
        self.gate_act, self.eps = gate_act, eps
        self.weight = torch.nn.Parameter(torch.ones(num_features))
        self.scale = torch.nn.Parameter(torch.full((num_features,), float(scale_init)))
        if next_norm:
            self.next_weight = torch.nn.Parameter(torch.ones(num_features))
        else:
            self.register_parameter("next_weight", None)

    def forward(self, x, y, gate=None, lengths=None):
        r = block_join(x, y, self.weight, gate=gate, gate_act=self.gate_act, scale=self.scale,
                       next_weight=self.next_weight, eps=self.eps, lengths=lengths)
        return r if self.next_weight is not None else r[0]
