"""Rotary positions: the rotation of queries and keys by their positions, and its frequencies."""
import math

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _host


def rotary_frequencies(rot_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, fast_turns=32.0, slow_turns=1.0,
                       device="cuda"):
    """The frequencies of the ``rot_dim / 2`` pairs that a rotation turns, in radians per position (float64 on ``device``), and
    the magnitude to rotate with: ``(freqs, magnitude)`` for ``rotary``, ``paged_kvcache_append`` and ``attention_paged_int8``.

    Pair i has ``base ** (-2 i / rot_dim)``.  ``scaling`` stretches a context of ``original_length`` positions by ``factor``:

    * ``"linear"``: all positions closer together, every frequency divided by ``factor``;
    * ``"base"``: a larger base, so that the slowest pair is divided by ``factor`` and the fastest stays as it is;
    * ``"parts"``: pairs that turn more than ``fast_turns`` times within ``original_length`` stay, those that turn less than
      ``slow_turns`` times are divided by ``factor``, the ones between in proportion; the magnitude is ``0.1 ln(factor) + 1``.
    """
    if rot_dim <= 0 or rot_dim % 16 != 0:
        raise ValueError(f"rot_dim must be a positive multiple of 16, got {rot_dim}")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be over 1 and factor at least 1")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    if scaling == "base" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freqs, magnitude = base ** (-2.0 * i / rot_dim), 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "parts":
        if original_length is None or not 0.0 <= slow_turns < fast_turns:
            raise ValueError('scaling="parts" needs original_length, and slow_turns below fast_turns')
        turns = original_length * freqs / (2.0 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        freqs = freqs * (keep + (1.0 - keep) / factor)
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f'scaling must be None, "linear", "base" or "parts", got {scaling!r}')
    return freqs.to(device), magnitude


class _Rotary(torch.autograd.Function):
    """The map is linear: its tangent goes through it, its gradient through the transposed one, and either of them may be differentiated again."""

    @staticmethod
    def forward(x, positions, freqs, interleaved, inverse, magnitude):
        return _host.native().rotary(x, positions, freqs, interleaved, inverse, magnitude)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, positions, freqs, *rest = inputs
        kept = (freqs, positions) if torch.is_tensor(positions) else (freqs,)
        ctx.save_for_backward(*kept)
        ctx.save_for_forward(*kept)
        ctx.rest = (None if torch.is_tensor(positions) else positions, *rest)

    @staticmethod
    def backward(ctx, grad):
        freqs, *positions = ctx.saved_tensors
        first, interleaved, inverse, magnitude = ctx.rest
        return rotary(grad, positions[0] if positions else first, freqs, interleaved=interleaved, inverse=not inverse, magnitude=magnitude), *[None] * 5

    @staticmethod
    def jvp(ctx, tangent, *_):
        freqs, *positions = ctx.saved_tensors
        first, interleaved, inverse, magnitude = ctx.rest
        return rotary(tangent, positions[0] if positions else first, freqs, interleaved=interleaved, inverse=inverse, magnitude=magnitude)


def rotary(x, positions, freqs, *, interleaved=False, inverse=False, magnitude=1.0):
    """Rotates x [Z, H, N, d] (fp16 or bf16; d 16, 32, 64, 128 or 256) by its positions; returns a new contiguous tensor.

    ``freqs``: float64 [pairs] radians per position (``rotary_frequencies``); a multiple of 8 pairs.  Pair i is the elements
    (i, i + pairs), or (2 i, 2 i + 1) with ``interleaved``; elements past 2 * pairs pass unchanged.
    ``positions``: an int (row n of every entry stands at positions + n), an int32 [Z] tensor (the first row's position of each
    entry) or an int32 [Z, N] tensor.  Angles are formed and reduced in fp64, so far positions keep theirs.
    ``inverse`` turns by the negative angle, times the same ``magnitude``: the transposed map.  Where x requires a gradient, it
    goes back through that; tangents of forward mode go through the map itself, and both can be differentiated again (frequencies and positions
    have neither).  A captured backward pass is captured with its forward pass, while no eager graph of x's leaves is alive.
    """
    if (x.requires_grad and torch.is_grad_enabled()) or _forward_ad._current_level >= 0:
        return _Rotary.apply(x, positions, freqs, interleaved, inverse, magnitude)
    return (_host._native or _host.native()).rotary(x, positions, freqs, interleaved, inverse, magnitude)
