"""Rotary positions with one or more axes: text, or time, height and width of images and video.

Pair i of a head's first ``2 * sum(sections)`` elements is turned by
``positions[axis(i)][token] * inv_freq[i]``; the first ``sections[0]`` pairs follow axis 0, the next
``sections[1]`` axis 1, and so on.  Pairs are elements (i, i + pairs), or neighbours when
``interleaved``.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import call_on

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}   # AMP_DTYPE_F32, AMP_DTYPE_BF16


def tensor_strides(t, name: str, device, dtype, T: int, D: int):
    """(token, head) stride in elements of a [T, heads, D] tensor whose last dimension is contiguous."""
    if t.dim() != 3 or t.dtype != dtype or t.device != device or t.shape[0] != T or t.shape[2] != D:
        raise ValueError(f"{name}: expected a {dtype} tensor [{T}, heads, {D}] on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    tok, head, inner = t.stride()
    # the stride of a dimension of one element says nothing
    if t.shape[1] <= 1:
        head = D
    if T <= 1:
        tok = max(1, t.shape[1]) * D
    if (D > 1 and inner != 1) or tok <= 0 or head <= 0:
        raise ValueError(f"{name}: the last dimension must be contiguous and the other strides "
                         f"positive, got {t.stride()}")
    return tok, head


def angle_args(positions, inv_freq, sections, device, T: int):
    """(positions, stride, axes, sections, inv_freq) for the C ABI, checked; the ctypes array of
    the sections must live until the call."""
    if positions.device != device or positions.dtype != torch.int32 \
            or positions.dim() not in (1, 2) or positions.shape[-1] != T \
            or (T > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions: expected int32 [{T}] or [axes, {T}] on {device}")
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    if inv_freq.device != device or inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 \
            or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq: expected a contiguous float32 vector on {device}")
    if sections is None and axes == 1:
        sections = (inv_freq.numel(),)
    if sections is None or len(sections) != axes or sum(sections) != inv_freq.numel():
        raise ValueError(f"sections {sections}: one count of pairs for each of {axes} axes, "
                         f"{inv_freq.numel()} (the entries of inv_freq) in all")
    stride = positions.stride(0) if positions.dim() == 2 and axes > 1 else T
    return positions.data_ptr(), stride, axes, (C.c_int32 * axes)(*sections), inv_freq.data_ptr()


def _rope(q, k, positions, inv_freq, sections, interleaved, out_q, out_k, backward):
    if q.dim() != 3 or not q.is_cuda or q.dtype not in _DTYPES:
        raise ValueError("q: expected a bf16 or float32 CUDA tensor [tokens, heads, head_dim]")
    T, Hq, D = q.shape
    dev = q.device
    angles = angle_args(positions, inv_freq, sections, dev, T)
    if out_q is None:
        out_q = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    if k is not None and out_k is None:
        out_k = torch.empty(k.shape, dtype=k.dtype, device=dev)
    strides, ptrs = [], []
    for x, name in ((q, "q"), (out_q, "out_q"), (k, "k"), (out_k if k is not None else None, "out_k")):
        strides += tensor_strides(x, name, dev, q.dtype, T, D) if x is not None else (D, D)
        ptrs.append(x.data_ptr() if x is not None else None)
    if out_q.shape != q.shape or (k is not None and out_k.shape != k.shape):
        raise ValueError("out_q and out_k must have the shapes of q and k")
    call_on(dev, "amp_rope_dev", *ptrs, _DTYPES[q.dtype], T, Hq, k.shape[1] if k is not None else 0,
            D, (C.c_int64 * 8)(*strides), *angles, 1 if interleaved else 0, 1 if backward else 0)
    return out_q, out_k


def rope_fwd(q, k, positions, inv_freq, sections=None, interleaved: bool = False, out_q=None,
             out_k=None):
    """Turns q [tokens, Hq, D] and k [tokens, Hk, D] (bf16 or fp32, any token and head strides; k
    may be None) and returns (q', k').  positions int32 [axes, tokens] (or [tokens]), inv_freq fp32
    [pairs], sections the pairs of each axis.  An output may be its input."""
    return _rope(q, k, positions, inv_freq, sections, interleaved, out_q, out_k, False)


def rope_bwd(dq, dk, positions, inv_freq, sections=None, interleaved: bool = False, out_q=None,
             out_k=None):
    """The gradients of rope_fwd's inputs from those of its outputs: the same turn, backwards."""
    return _rope(dq, dk, positions, inv_freq, sections, interleaved, out_q, out_k, True)
