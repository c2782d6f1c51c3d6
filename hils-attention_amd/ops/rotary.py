"""Rotary positions by position: any position per token, half or interleaved pairs, part of the head, frequencies scaled
for long contexts.

The reference rotates by tables that its model lays out by row (models/FlashHiLS/hils_attention.py:466-488,
ops/rope_tilelang_fp32.py); drafted tokens, packed sequences and slices of a cache have positions of their own.
"""
import math

import torch

from . import _cabi
from ._native_op import NativeOp


class _RotaryEmbedding(NativeOp):
    @staticmethod
    def native(q, k, positions, first, inv_freq, interleaved, scale):
        return _cabi.host().rotary_embedding(q, k, positions, first, inv_freq, interleaved, scale)

    @staticmethod
    def forward(ctx, *args):
        return NativeOp.record(ctx, _RotaryEmbedding.native, args)


def rotary_embedding(q, k, positions, inv_freq, interleaved=False, scale=1.0):
    """q (B,T,H_q,D), k (B,T,H_kv,D) or None, bf16, any strides -> rotated copies (q_out, k_out), bf16.

    The first ``2 * len(inv_freq)`` features of a head are pairs, features i and i + len(inv_freq), or with ``interleaved``
    2i and 2i + 1; a pair turns by ``positions * inv_freq[i]`` and is multiplied by ``scale``; the other features pass
    through.  ``positions``: int32 or int64, (T,) or (B,T), or an int, the position of the first token.  ``inv_freq``: fp32
    or fp64 on the GPU (``rotary_frequencies``).  Angles and rotation are fp64, so far positions keep their precision; the
    result is rounded to bf16 by way of fp32: half a step of bf16 and at most 2^-24 more.  Differentiable in q and k."""
    first = 0
    if not isinstance(positions, torch.Tensor):
        first, positions = int(positions), None
    return _RotaryEmbedding.apply(q, k, positions, first, inv_freq, bool(interleaved), float(scale))


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=None, high=None,
                       device="cuda"):
    """(inv_freq (rotary_dim / 2,) fp64, scale) for ``rotary_embedding``: base^(-2i / rotary_dim), scaled for contexts
    ``factor`` times the length that a model was trained on:

    * ``None``          as they are;
    * ``"linear"``      all divided by ``factor`` (positions interpolated);
    * ``"ntk"``         base times factor^(d / (d - 2)): the slowest pair divided by ``factor``, the fastest kept;
    * ``"yarn"``        pairs that turn more than ``high`` (32) times over ``original_length`` kept, fewer than ``low`` (1)
                        divided by ``factor``, between them a ramp in the number of turns; scale 0.1 ln(factor) + 1;
    * ``"wavelength"``  the same ramp between ``low`` (1) and ``high`` (4) turns, scale 1.

    The ramp is linear in the number of turns, as the method's formula has it.  A checkpoint trained with a ramp that is
    linear in the pair's number i, which also goes by the name of yarn, has other frequencies between the two ends: hand
    ``rotary_embedding`` that model's own ``inv_freq``."""
    rotary_dim = int(rotary_dim)
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (base > 1 and factor >= 1):
        raise ValueError(f"base must be above 1 and factor at least 1, got {base} and {factor}")
    power = -torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs two pairs at least")
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** power, 1.0
    inv_freq = base ** power
    if scaling is None:
        return inv_freq, 1.0
    if scaling == "linear":
        return inv_freq / factor, 1.0
    if scaling not in ("yarn", "wavelength"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not original_length or original_length <= 0:
        raise ValueError(f"{scaling} scaling needs original_length, the context that the frequencies were trained on")
    low = 1.0 if low is None else float(low)
    high = (32.0 if scaling == "yarn" else 4.0) if high is None else float(high)
    if not 0 <= low < high:
        raise ValueError(f"low ({low}) must be below high ({high})")
    keep = ((original_length * inv_freq / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return inv_freq * keep + inv_freq / factor * (1 - keep), 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
