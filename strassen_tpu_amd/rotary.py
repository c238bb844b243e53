"""Rotary positions at positions of the program's own, on the kernels of ``csrc/rotary.hip``.

The GEMM's ``qk_norm_rope`` epilogue and ``paged_write`` rotate by tables whose row is the token's index in its
sequence or cache. ``rotary`` takes the positions themselves and works the angles out: for tokens of a cache
from which others were evicted, contexts too long for a table, heads in other layouts or rotated in part."""

from __future__ import annotations

import math

import torch

from . import _lib

__all__ = ["rotary", "rotary_frequencies", "ROTARY_SCALINGS"]

ROTARY_SCALINGS = ("linear", "ntk", "yarn", "bands")


def rotary_frequencies(rotary_dim, theta=1e6, *, scaling=None, factor=1.0, original_context=None, fast=None, slow=None,
                       device=None):
    """Angles per position of ``rotary_dim / 2`` pairs (float64) and the amplitude, for ``rotary``:
    ``theta ** (-2 i / rotary_dim)`` and 1. ``scaling`` stretches them for contexts ``factor`` times as long as the
    ``original_context`` that a model was trained on:

    * ``"linear"`` (position interpolation): every angle divided by ``factor``;
    * ``"ntk"``: the base becomes ``theta * factor ** (d / (d - 2))``, which leaves the fastest pair as it
      was and divides the slowest one's angle by ``factor``;
    * ``"yarn"``: pairs that turn at least ``fast`` (32) times over the original context stay, those that turn at most
      ``slow`` (1) times are divided by ``factor``, with a linear ramp over the pairs between (from the pair
      below to the pair above); amplitude ``0.1 ln(factor) + 1``;
    * ``"bands"``: the same with a ramp that is linear in the turns, ``fast`` 4 and ``slow`` 1; amplitude 1."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    half = torch.arange(rotary_dim // 2, dtype=torch.float64)
    frequencies = theta ** (-2 * half / rotary_dim)
    if scaling is None:
        if factor != 1.0:
            raise ValueError("factor= goes with scaling=")
        return frequencies.to(device), 1.0
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}; expected one of {ROTARY_SCALINGS}")
    if not (factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling == "linear":
        return (frequencies / factor).to(device), 1.0
    if scaling == "ntk":
        if rotary_dim == 2:  # one pair, the fastest
            return frequencies.to(device), 1.0
        base = theta * factor ** (rotary_dim / (rotary_dim - 2))
        return (base ** (-2 * half / rotary_dim)).to(device), 1.0
    if original_context is None or original_context <= 0:
        raise ValueError(f"scaling={scaling!r} needs original_context=, the tokens that the model was trained on")
    if scaling == "yarn" and theta <= 1:
        raise ValueError(f"scaling='yarn' needs theta above 1, got {theta}")
    fast = fast if fast is not None else 32.0 if scaling == "yarn" else 4.0
    slow = 1.0 if slow is None else slow
    if not fast > slow > 0:
        raise ValueError(f"fast={fast} must be above slow={slow}, and both positive")
    if scaling == "bands":
        turns = original_context * frequencies / (2 * math.pi)
        stays = ((turns - slow) / (fast - slow)).clamp(0, 1)
        return (frequencies * stays + frequencies / factor * (1 - stays)).to(device), 1.0

    def pair(turns):  # the pair that turns so often over the original context
        return rotary_dim * math.log(original_context / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(0, math.floor(pair(fast))), min(rotary_dim - 1, math.ceil(pair(slow)))
    stretched = ((half - low) / max(high - low, 1e-3)).clamp(0, 1)
    return (frequencies * (1 - stretched) + frequencies / factor * stretched).to(device), 0.1 * math.log(factor) + 1.0


def rotary(x, positions, frequencies, *, interleaved=False, amplitude=1.0, norm=None, eps=1e-6, out=None):
    """Heads ``x [tokens, heads, head_dim]`` (bf16 or float32, any strides) rotated by their ``positions [tokens]``
    (int32 or int64): pair ``i`` of a head by ``positions * frequencies[i]`` radians, times
    ``amplitude``. The first ``2 * len(frequencies)`` values of a head are rotated, the others copied; a pair is
    ``(i, i + len(frequencies))``, with ``interleaved`` ``(2 i, 2 i + 1)``. ``norm [head_dim]`` RMS-normalises the
    whole head and scales it first (``eps``).

    Query and key heads that are columns of one projection are one ``x``. Angles are reduced in 64 bits from
    ``frequencies`` float64 (or float32, taken as they are), so that far positions lose nothing; the rest is FP32
    with one rounding. Rows of negative position (a plan's rows of no admitted request) are zero in a new result and left
    as they were in ``out``, which is ``x`` itself or shares no memory with it, and none with the other tensors. ``head_dim`` up
    to 1024, up to 2^20 tokens. No gradients.

    Heads whose rotated halves and width are whole runs of 16 bytes (8 bf16 values) at aligned places, behind a norm also a power
    of two wide, run at what memory gives; others take some three times as long."""
    return _lib.host().rotary(x, positions, frequencies, interleaved, amplitude, norm, eps, out)
