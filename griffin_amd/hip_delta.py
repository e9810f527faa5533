"""The gated delta rule on the GPU: a gated linear recurrence like the RG-LRU's, whose state is a matrix for each head,

    S_t = a_t (I - beta_t k_t k_t') S_{t-1} + beta_t k_t v_t',    o_t = scale S_t' q_t,    a_t = exp(log_decay_t)

over ``rglru_hip_gated_delta_*`` of librglru_hip.so.  Masks and carried state follow ``hip_rglru``; the reference has no
counterpart.  There is no CPU fallback here: the operators raise when the library or a GPU is missing.
"""

from __future__ import annotations

from torch import Tensor

from . import _lib


def _scale(scale: float | None, q: Tensor) -> float:
    return float(max(q.size(-1), 1)) ** -0.5 if scale is None else float(scale)


def hip_gated_delta(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, h0: Tensor | None = None,
                    scale: float | None = None, reset_mask: Tensor | None = None,
                    active_mask: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """The recurrence over whole sequences: returns ``(o [B, T, HV, V] in v.dtype, final state [B, HV, K, V] in fp32)``.

    ``q``, ``k`` [B, T, H, K] (K up to 128) and ``v`` [B, T, HV, V], all float32 or all bfloat16; ``log_decay`` and ``beta``
    [B, T, HV], float32 or bfloat16 each.  HV is a multiple of H: value head h reads key head ``h // (HV // H)``.  Views whose last
    axis is contiguous are read in place (the parts of one projection, for instance).  ``h0`` [B, HV, K, V] or None (zeros);
    ``scale``: K ** -0.5 by default.  Log decays are at most 0 by meaning; below -1e4 (minus infinity among them) they discard the
    history.  Keys of unit length and ``beta`` in [0, 2] keep the state bounded.

    ``reset_mask`` [B, T]: tokens that start a document (the history in front of them is discarded).  ``active_mask`` [B, T]: tokens
    that count; the others leave the state as it is, give zeros and receive zero gradients, whatever they hold.  Among the
    active tokens a NaN or an infinity may reach all outputs of its chunk of 64 tokens and those behind it, in gradients those in front
    of it.  Where the first active token of a chunk starts a document, the chunk takes nothing from what lies in front of it, a
    state of NaN included, and hands no gradient on to it.

    Products are exact to fp32 for float32 operands and to 2^-17 for what is computed between them from bfloat16 ones, relative to their terms:
    what the keys of a chunk all but erase (the gradient of ``h0`` behind many parallel keys) is known to that part of what it was, not
    of what is left.

    Differentiable (first order) in q, k, v, log_decay, beta and h0, through both results.
    """
    native = _lib.native()
    for name, mask in (("reset_mask", reset_mask), ("active_mask", active_mask)):
        if mask is not None and mask.shape != q.shape[:2]:
            raise ValueError(f"{name} must have shape {tuple(q.shape[:2])}, got {tuple(mask.shape)}")
    reset_mask, active_mask = (None if m is None else m.to(device=q.device) for m in (reset_mask, active_mask))
    flags = None if reset_mask is None and active_mask is None else native.pack_flags(reset_mask, active_mask)
    return native.gated_delta(q, k, v, log_decay, beta, h0, flags, _scale(scale, q))


def hip_gated_delta_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, state: Tensor,
                         scale: float | None = None, flags: Tensor | None = None) -> Tensor:
    """One token a row, without gradients: ``state`` [B, HV, K, V] fp32 is updated in place; returns o [B, HV, V] in v.dtype.

    ``q``, ``k`` [B, H, K], ``v`` [B, HV, V], ``log_decay`` and ``beta`` [B, HV] as for ``hip_gated_delta``; ``flags`` [B]: one byte a
    row, bit 0 = the token starts a document, bit 1 = the row has no token (its state stays as it is, its output is zero)."""
    return _lib.native().gated_delta_step(q, k, v, log_decay, beta, state, flags, _scale(scale, q))
