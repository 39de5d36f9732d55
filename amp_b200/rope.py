"""Rotary positions with one or more axes: text, or time, height and width of images and video.

Pair i of a head's first ``2 * sum(sections)`` elements is turned by
``positions[axis(i)][token] * inv_freq[i]``; the first ``sections[0]`` pairs follow axis 0, the next
``sections[1]`` axis 1, and so on (at most 4 axes).  Pairs are elements (i, i + pairs), or neighbours
when ``interleaved``.  No counterpart in the reference.
"""
from __future__ import annotations

from ._lib import ops


def rope_fwd(q, k, positions, inv_freq, sections=None, interleaved: bool = False, out_q=None,
             out_k=None):
    """Turns q [tokens, Hq, D] and k [tokens, Hk, D] (bf16 or fp32, any token and head strides; k
    may be None) and returns (q', k').  positions int32 [axes, tokens] (an expanded row is taken
    as it is) or [tokens], contiguous along the tokens; inv_freq fp32 [pairs], sections the pairs of
    each axis (with one axis: None).  An output may be its input, and shares no memory with others."""
    return ops().rope(q, k, positions, inv_freq, sections, interleaved, out_q, out_k, False)


def rope_bwd(dq, dk, positions, inv_freq, sections=None, interleaved: bool = False, out_q=None,
             out_k=None):
    """The gradients of rope_fwd's inputs from those of its outputs: the same turn, backwards."""
    return ops().rope(dq, dk, positions, inv_freq, sections, interleaved, out_q, out_k, True)
