"""The operators of a block around a selective state space on the GPU: the scan, whose channels carry a few numbers each that the tokens themselves
decide how to keep, write and read,

    s_t = softplus(dt_t + dt_bias),   h_t[w, n] = exp(s_t[w] A[w, n]) h_{t-1}[w, n] + s_t[w] u_t[w] B_t[n]
    y_t[w] = (sum over n of C_t[n] h_t[w, n] + D[w] u_t[w]) silu(z_t[w])

and the short causal convolution with an activation in front of it, for whole sequences and for single tokens, over ``rglru_hip_selective_*`` and
``rglru_hip_short_conv_*`` of librglru_hip.so.  Masks and carried state follow ``hip_rglru``; the reference has no counterpart.  There is no CPU
fallback here: the operators raise when the library or a GPU is missing.
"""

from __future__ import annotations

from torch import Tensor

from . import _lib

_ACTIVATIONS = {None: 0, "silu": 1}                          # RGLRU_ACT_* of the C ABI


def _flags(native, like: Tensor, reset_mask: Tensor | None, active_mask: Tensor | None) -> Tensor | None:
    for name, mask in (("reset_mask", reset_mask), ("active_mask", active_mask)):
        if mask is not None and mask.shape != like.shape[:2]:
            raise ValueError(f"{name} must have shape {tuple(like.shape[:2])}, got {tuple(mask.shape)}")
    if reset_mask is None and active_mask is None:
        return None
    return native.pack_flags(*(None if m is None else m.to(device=like.device) for m in (reset_mask, active_mask)))


def _activation(name: str, activation: str | None) -> int:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{name} knows the activations None and 'silu', got {activation!r}")
    return _ACTIVATIONS[activation]


def hip_selective_scan(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None, z: Tensor | None = None,
                       dt_bias: Tensor | None = None, h0: Tensor | None = None, softplus: bool = True, reset_mask: Tensor | None = None,
                       active_mask: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """The scan over whole sequences: returns ``(y [B, T, W] in u.dtype, final state [B, W, N] in fp32)``.

    ``u``, ``dt`` and the gate ``z`` (None: no gate) [B, T, W], ``B`` and ``C`` [B, T, G, N] (N up to 64), all float32 or all bfloat16; channel w reads
    group ``w // (W // G)``.  ``A`` [W, N], finite and negative by meaning; ``D`` (None: zeros) and ``dt_bias`` (None: zeros) [W], float32 or
    bfloat16 each, float32 as they are.  ``softplus=False`` takes ``dt + dt_bias`` itself for the step size.  ``h0`` [B, W, N] or None (zeros).  Views whose
    last axis is contiguous are read in place (the parts of one projection, for instance).

    ``reset_mask`` [B, T]: tokens that start a document (the history in front of them is discarded, whatever it is).  ``active_mask`` [B, T]: tokens that
    count; the others leave the state as it is, give zeros and receive zero gradients, whatever they hold.

    States, sums and step sizes are fp32; a result is rounded once.  A backward pass needs the state in front of every 16 tokens, ``N / 4`` bytes a
    token and channel, which the forward pass keeps.  Differentiable (first order) in all operands but the masks, through both results."""
    native = _lib.native()
    return native.selective_scan(u, dt, A, B, C, D, z, dt_bias, h0, _flags(native, u, reset_mask, active_mask), softplus)


def hip_selective_step(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None = None, z: Tensor | None = None,
                       dt_bias: Tensor | None = None, softplus: bool = True, flags: Tensor | None = None) -> Tensor:
    """One token a row, without gradients: ``state`` [B, W, N] fp32 is updated in place; returns y [B, W] in u.dtype.

    ``u``, ``dt``, ``z`` [B, W], ``B``, ``C`` [B, G, N], the others as for ``hip_selective_scan``; ``flags`` [B]: one byte a row, bit 0 = the token
    starts a document, bit 1 = the row has no token (its state stays as it is, its output is zero)."""
    return _lib.native().selective_step(u, dt, A, B, C, state, D, z, dt_bias, flags, softplus)


def hip_short_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, state: Tensor | None = None, activation: str | None = None,
                   reset_mask: Tensor | None = None, active_mask: Tensor | None = None, need_state: bool = True) -> tuple[Tensor, Tensor | None]:
    """``act(causal depthwise convolution)`` of ``x`` [B, T, W]: returns ``(y [B, T, W], new_state [B, K - 1, W])``, float32 or bfloat16.

    ``weight`` [W, 1, K] (K up to 4) and ``bias`` [W] of a depthwise ``nn.Conv1d``; ``state`` [B, K - 1, W]: the inputs in front of the first token, the newest
    last (None: zeros); ``activation``: None or "silu".  ``x`` may be a view whose last axis is contiguous.  Masks as for ``hip_selective_scan``, holes
    included: a document starts with an empty window, inactive tokens stay out of it and give zeros.  ``new_state``, the window behind the last
    token, is a cache for the next call and carries no gradient (None without ``need_state``); ``y`` is differentiable in x, weight, bias and state."""
    native = _lib.native()
    code = _activation("hip_short_conv", activation)
    return native.short_conv(x, weight, bias, state, _flags(native, x, reset_mask, active_mask), code, need_state)


def hip_short_conv_step(x: Tensor, weight: Tensor, bias: Tensor | None, state: Tensor, activation: str | None = None,
                        flags: Tensor | None = None) -> Tensor:
    """One token a row, ``x`` [B, W], without gradients: ``state`` [B, K - 1, W] in x.dtype is updated in place; returns y [B, W].  ``flags`` as for
    ``hip_selective_step``."""
    code = _activation("hip_short_conv_step", activation)
    return _lib.native().short_conv_step(x, weight, bias, state, flags, code)
