"""Frequencies of rotary positions, with the usual scalings for long contexts, and the
rotation's gradient.

`rope_frequencies` gives what `cuda_ops.rope` (dsr_rope) takes: one angular
frequency per rotated pair, in 64 bits, and the amplitude of the rotated columns.
`Rotation` is that call for tensors that require a gradient.
"""
from __future__ import annotations

import math

import torch

from .cuda_ops import ValidationError, _status, extension

SCALINGS = ("none", "linear", "ntk", "yarn")


def rope_frequencies(dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_context: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(f64[dim // 2] frequencies on the CPU, amplitude) of `dim` rotated columns.

    none:   base^(-2i/dim)
    linear: the same over `factor` (positions interpolated)
    ntk:    base grown by factor^(dim/(dim-2)): the slowest pair is interpolated by
            `factor`, the fastest stays
    yarn:   pairs that turn more than `beta_fast` times over `original_context` stay,
            those below `beta_slow` turns are interpolated by `factor`, a linear ramp
            between them; amplitude 0.1 ln(factor) + 1
    """
    if isinstance(dim, bool) or not isinstance(dim, int) or not 2 <= dim <= 512 or dim % 2:
        raise ValidationError("rotated columns must be an even integer in [2, 512]")
    if scaling not in SCALINGS:
        raise ValidationError(f"rotary scaling must be one of {', '.join(SCALINGS)}")
    if not (math.isfinite(base) and base > 1 and math.isfinite(factor) and factor >= 1):
        raise ValidationError("rotary base must exceed 1 and the scaling factor must be at least 1")
    pairs = dim // 2
    if scaling == "ntk":
        if dim == 2:
            raise ValidationError("ntk scaling needs at least two pairs")
        base = base * factor ** (dim / (dim - 2))
    frequencies = float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    if scaling == "linear":
        return frequencies / factor, 1.0
    if scaling != "yarn":
        return frequencies, 1.0
    if not (original_context > 0 and beta_fast > beta_slow > 0):
        raise ValidationError("yarn needs a positive original context and beta_fast > beta_slow > 0")

    def pair_of(turns):  # the (fractional) pair that turns so often over the original context
        return pairs * math.log(original_context / (turns * 2 * math.pi)) / math.log(base)

    low = max(math.floor(pair_of(beta_fast)), 0)
    high = min(math.ceil(pair_of(beta_slow)), dim - 1)
    ramp = ((torch.arange(pairs, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return frequencies * (1 - ramp) + frequencies / factor * ramp, 0.1 * math.log(factor) + 1.0


class Rotation(torch.autograd.Function):
    """cuda_ops.rope into new tensors.  The rotation is linear, so its gradient is the
    transposed one: the same amplitude, the angles negated; padding rows pass as they are."""

    @staticmethod
    def forward(ctx, positions, frequencies, offsets, interleaved, mscale, inverse, check, *tensors):
        out = [t.detach().clone() for t in tensors]
        status = extension().rope(list(tensors), out, positions, frequencies, offsets, interleaved, mscale=mscale,
                                  inverse=inverse)
        if check:
            _status(status)
        ctx.save_for_backward(positions, frequencies)
        ctx.settings = offsets, interleaved, mscale, inverse
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(o for o, needed in zip(out, ctx.needs_input_grad[7:]) if not needed))
        return tuple(out)

    @staticmethod
    def backward(ctx, *grads):
        positions, frequencies = ctx.saved_tensors
        offsets, interleaved, mscale, inverse = ctx.settings
        at = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[7 + i]]
        result = [None] * len(grads)
        if at:  # the positions have passed the forward's check
            turned = Rotation.apply(positions, frequencies, [offsets[i] for i in at], [interleaved[i] for i in at],
                                    mscale, not inverse, False, *(grads[i].contiguous() for i in at))
            for i, g in zip(at, turned):
                result[i] = g
        return (None,) * 7 + tuple(result)
