"""Rotary positions: tables for short and scaled long contexts, and the rotation with its gradient.

The reference leaves RoPE to the Hugging Face model around its packed linears.  Here ``rope_tables`` builds the
float32 cos / sin tables that every kernel of this package takes (``[max_len, rotary_dim / 2]``, angles in 64
bits, a scaling's gain folded in), and ``rope`` rotates q and k in one launch (include/epq_paged.h, epq_rope).
"""
import math

import torch

from . import _native

SCALINGS = ("none", "linear", "ntk", "bands", "yarn")


def rope_frequencies(rotary_dim, theta=1.0e4, scaling="none", factor=1.0, original_max=8192, low=1.0, high=4.0,
                     beta_fast=32.0, beta_slow=1.0, gain=None):
    """(frequencies [rotary_dim / 2] in float64, gain) of a rotary embedding ``theta ** (-2 j / rotary_dim)``.

    ``scaling`` stretches the positions that a model was trained on (``original_max``) by ``factor``:

    * ``"linear"``: every frequency divided by the factor;
    * ``"ntk"``: theta raised to ``theta * factor ** (r / (r - 2))``, so the lowest frequency is divided by the
      factor and the highest stays;
    * ``"bands"``: by the turns that a pair makes over ``original_max`` positions: fewer than ``low`` are divided
      by the factor, more than ``high`` stay, a linear ramp between them;
    * ``"yarn"``: a linear ramp over the pairs' index between those that make ``beta_fast`` and ``beta_slow``
      turns; the tables are multiplied by ``gain`` (default ``0.1 ln(factor) + 1``)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"epure: rotary_dim must be even and positive (got {rotary_dim})")
    if scaling not in SCALINGS:
        raise ValueError(f"epure: scaling must be one of {SCALINGS} (got {scaling!r})")
    if factor <= 0 or theta <= 0:
        raise ValueError(f"epure: theta and factor must be positive (got {theta}, {factor})")
    if scaling == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    j = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    f = theta ** (-j / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        if not high > low:
            raise ValueError(f"epure: high must be above low (got {low}, {high})")
        keep = ((original_max * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / factor
    elif scaling == "yarn":
        at = [rotary_dim * math.log(original_max / (n * 2 * math.pi)) / (2 * math.log(theta))
              for n in (beta_fast, beta_slow)]
        first, final = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
        ramp = ((j / 2 - first) / max(final - first, 1e-3)).clamp(0, 1)
        f = (1 - ramp) * f + ramp * f / factor
        if gain is None:
            gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return f, 1.0 if gain is None else float(gain)


def rope_tables(rotary_dim, max_len, device="cuda", **kw):
    """Float32 ``(cos, sin)`` ``[max_len, rotary_dim / 2]`` (keywords as ``rope_frequencies``)."""
    if max_len < 1:
        raise ValueError(f"epure: max_len must be positive (got {max_len})")
    f, gain = rope_frequencies(rotary_dim, **kw)
    angle = torch.arange(max_len, dtype=torch.float64, device=device)[:, None] * f.to(device)
    return (gain * angle.cos()).float(), (gain * angle.sin()).float()


def _calls():
    return _native.tensor_calls or _native.load_tensor_calls()


class _RopeFn(torch.autograd.Function):
    """The gradient of a rotation is the rotation back: dx = R^T dy."""

    @staticmethod
    def forward(ctx, pos, cos, sin, interleaved, inverse, q, k):
        ctx.save_for_backward(pos, cos, sin)
        ctx.how = (interleaved, inverse)
        return _calls().rope(q, k, pos, cos, sin, interleaved, inverse, None, None)

    @staticmethod
    def backward(ctx, dq, dk=None):
        # by rope() itself, so that a gradient's gradient is one too
        pos, cos, sin = ctx.saved_tensors
        interleaved, inverse = ctx.how
        dq = dq if dq.stride(-1) == 1 else dq.contiguous()
        dk = dk if dk is None or dk.stride(-1) == 1 else dk.contiguous()
        got = rope(dq, dk, pos, cos, sin, interleaved, not inverse)
        return (None,) * 5 + ((got, None) if dk is None else got)


def rope(q, k, pos, cos, sin, interleaved=False, inverse=False, out=None):
    """Rotates q (and k, unless None) ``[rows, heads, head_dim]`` by their positions ``pos`` [rows] (int64).

    The first ``rotary_dim`` values of every head (the tables' width times two) turn, pairs ``(j, j + r / 2)``, or
    ``(2j, 2j + 1)`` with ``interleaved``; the others are copied.  float32, float16 or bfloat16; rows and heads
    may be strided.  ``inverse`` turns back (for a gradient: ``dq, dk = rope(dy_q, dy_k, ..., inverse=True)``);
    autograd does so by itself (for q and k; tables that require a gradient are refused, and so are tensors with
    a forward-mode tangent).  ``out=(q_out, k_out)`` writes there, in place where they are q and k; it records
    nothing for autograd, so with grad mode on, tensors that require a gradient are refused.  Returns ``(q', k')``, or ``q'`` alone without k."""
    if out is not None:
        q_out, k_out = out if k is not None else (out if torch.is_tensor(out) else out[0], None)
        return _calls().rope(q, k, pos, cos, sin, interleaved, inverse, q_out, k_out)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if cos.requires_grad or sin.requires_grad:
            raise RuntimeError("epure: rope has no gradient with respect to cos and sin; detach them")
        return _RopeFn.apply(pos, cos, sin, interleaved, inverse, q, k)
    return _calls().rope(q, k, pos, cos, sin, interleaved, inverse, None, None)
