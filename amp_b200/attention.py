"""FlashAttention-2: host-side mirror of kernels/flash_attn.cuh, its backward, and
both over packed sequences of different lengths.

``launch_flash_attn_bf16(Q, K, V, O, lse, B, S_q, S_kv, cfg)`` mirrors
``AMP::launch_flash_attn_bf16`` (kernels/flash_attn.cuh:50-58) with the same
AttnCfg fields (flash_attn.cuh:26-36).  The tile fields Br/Bc are accepted for
source compatibility; the sm_100a kernel always uses 128x128 tiles.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from ._lib import call, call_on, lib


@dataclass
class AttnCfg:
    num_q_heads: int = 1
    num_kv_heads: int = 1
    head_dim: int = 128
    causal: bool = True
    scale: float = 0.0      # 0 -> 1/sqrt(head_dim)
    Br: int = 32
    Bc: int = 64


def _check(t, shape, name, dtype=torch.bfloat16):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous() or tuple(t.shape) != shape:
        raise ValueError(f"{name}: expected contiguous {dtype} CUDA tensor {shape}, "
                         f"got {t.dtype} {tuple(t.shape)}")


def launch_flash_attn_bf16(Q, K, V, O, lse, B: int, S_q: int, S_kv: int, cfg: AttnCfg) -> None:
    Hq, Hkv, D = cfg.num_q_heads, cfg.num_kv_heads, cfg.head_dim
    _check(Q, (B, Hq, S_q, D), "Q")
    _check(K, (B, Hkv, S_kv, D), "K")
    _check(V, (B, Hkv, S_kv, D), "V")
    _check(O, (B, Hq, S_q, D), "O")
    if lse is not None:
        _check(lse, (B, Hq, S_q), "lse", torch.float32)
    call("amp_flash_attn_fwd_bf16_dev", Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(),
         lse.data_ptr() if lse is not None else None, B, Hq, Hkv, S_q, S_kv, D,
         1 if cfg.causal else 0, float(cfg.scale), torch.cuda.current_stream(Q.device).cuda_stream)


def flash_attn_fwd(q, k, v, causal: bool = True, scale: float = 0.0):
    """Convenience form: returns (O, lse) for [B,H,S,D] bf16 CUDA tensors."""
    B, Hq, S_q, D = q.shape
    Hkv, S_kv = k.shape[1], k.shape[2]
    O = torch.empty_like(q)
    lse = torch.empty(B, Hq, S_q, dtype=torch.float32, device=q.device)
    launch_flash_attn_bf16(q, k, v, O, lse, B, S_q, S_kv,
                           AttnCfg(Hq, Hkv, D, causal, scale))
    return O, lse


def flash_attn_bwd(q, k, v, o, do, lse, causal: bool = True, scale: float = 0.0,
                   workspace: torch.Tensor | None = None):
    """Backward of flash_attn_fwd: returns (dQ, dK, dV) from the forward's q, k, v,
    o, lse and the upstream gradient do (all [B,H,S,D] bf16 CUDA tensors; lse fp32)."""
    B, Hq, S_q, D = q.shape
    Hkv, S_kv = k.shape[1], k.shape[2]
    _check(q, (B, Hq, S_q, D), "q")
    _check(k, (B, Hkv, S_kv, D), "k")
    _check(v, (B, Hkv, S_kv, D), "v")
    _check(o, (B, Hq, S_q, D), "o")
    _check(do, (B, Hq, S_q, D), "do")
    _check(lse, (B, Hq, S_q), "lse", torch.float32)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws_b = int(lib().amp_flash_attn_bwd_workspace_bytes(B, Hq, S_q))
    ws = workspace if workspace is not None else torch.empty(ws_b, dtype=torch.uint8,
                                                             device=q.device)
    call("amp_flash_attn_bwd_bf16_dev", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
         do.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, Hq, Hkv,
         S_q, S_kv, D, 1 if causal else 0, float(scale), ws.data_ptr(), ws.numel(),
         torch.cuda.current_stream(q.device).cuda_stream)
    return dq, dk, dv


def _packed(t, name: str, tokens, heads, D, device, strides: list):
    """A bf16 [tokens, heads, D] CUDA tensor on `device` whose last dimension is contiguous
    and whose other strides are positive multiples of 8 (a view into a fused projection,
    for example); appends its token and head stride.  Returns its pointer."""
    if t.dim() != 3 or t.dtype != torch.bfloat16 or not t.is_cuda or t.device != device \
            or t.shape[1] != heads or t.shape[2] != D or (tokens is not None and t.shape[0] != tokens):
        raise ValueError(f"{name}: expected a bf16 tensor [{'tokens' if tokens is None else tokens}"
                         f", {heads}, {D}] on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    tok, head, inner = t.stride()
    # the stride of a dimension of one element says nothing
    if t.shape[1] <= 1:
        head = D
    if t.shape[0] <= 1:
        tok = heads * D
    if inner != 1 or tok <= 0 or head <= 0 or tok % 8 or head % 8:
        raise ValueError(f"{name}: the last dimension must be contiguous and the other strides "
                         f"positive multiples of 8 elements, got {t.stride()}")
    strides += (tok, head)
    return t.data_ptr()


def _offsets(cu, name: str, device):
    if not cu.is_cuda or cu.device != device or cu.dtype != torch.int32 or cu.dim() != 1 \
            or not cu.is_contiguous() or cu.numel() < 2:
        raise ValueError(f"{name}: expected a contiguous int32 tensor [sequences + 1] on {device}")
    return cu.data_ptr()


def _varlen_shapes(q, k, v, cu_seqlens, cu_seqlens_kv):
    if q.dim() != 3 or k.dim() != 3 or not q.is_cuda:
        raise ValueError("q, k, v: expected packed CUDA tensors [tokens, heads, head_dim]")
    cu_kv = cu_seqlens if cu_seqlens_kv is None else cu_seqlens_kv
    if cu_kv.numel() != cu_seqlens.numel():
        raise ValueError("cu_seqlens and cu_seqlens_kv must have the same number of entries")
    return cu_kv, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]


def _workspace(workspace, nbytes: int, device):
    if workspace is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if not workspace.is_cuda or workspace.device != device or workspace.dtype != torch.uint8 \
            or not workspace.is_contiguous() or workspace.numel() < nbytes:
        raise ValueError(f"workspace: expected a contiguous uint8 tensor of >= {nbytes} bytes "
                         f"on {device}")
    return workspace


def _check_varlen_lse(lse, Hq: int, tokens: int, device):
    if lse.dtype != torch.float32 or tuple(lse.shape) != (Hq, tokens) or lse.device != device \
            or not lse.is_contiguous():
        raise ValueError(f"lse: expected a contiguous float32 tensor {(Hq, tokens)} on {device}")


def flash_attn_varlen_fwd(q, k, v, cu_seqlens, cu_seqlens_kv=None, causal: bool = True,
                          scale: float = 0.0, out=None, lse=None, workspace=None):
    """Attention over packed sequences: returns (O [tokens, Hq, D], lse [Hq, tokens]).

    q [tokens, Hq, D], k and v [kv tokens, Hkv, D]: bf16, any token and head strides that are
    multiples of 8 elements, so that parts of one fused projection are taken as they are.
    Sequence b is rows cu_seqlens[b] .. cu_seqlens[b+1] of q, and of k and v by cu_seqlens_kv
    (int32 CUDA tensors; cu_seqlens when None).  Under the causal mask the last query sees every
    key of its sequence.  A query that sees none gets O = 0 and lse = -inf.  Rows that belong to
    no sequence are not written: in outputs allocated here they are unspecified.  A workspace
    (uint8, amp_flash_attn_varlen_workspace_bytes) must not be shared by calls that may overlap."""
    cu_kv, T, Tk, Hq, Hkv, D = _varlen_shapes(q, k, v, cu_seqlens, cu_seqlens_kv)
    dev, strides = q.device, []
    ptr = [_packed(q, "q", T, Hq, D, dev, strides), _packed(k, "k", Tk, Hkv, D, dev, strides),
           _packed(v, "v", Tk, Hkv, D, dev, strides)]
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    ptr.append(_packed(out, "out", T, Hq, D, dev, strides))
    if lse is None:
        lse = torch.empty(Hq, T, dtype=torch.float32, device=dev)
    else:
        _check_varlen_lse(lse, Hq, T, dev)
    B = cu_seqlens.numel() - 1
    ws = _workspace(workspace, lib().amp_flash_attn_varlen_workspace_bytes(B), dev)
    call_on(dev, "amp_flash_attn_varlen_fwd_bf16_dev", *ptr, lse.data_ptr(),
            _offsets(cu_seqlens, "cu_seqlens", dev), _offsets(cu_kv, "cu_seqlens_kv", dev), B, T, Tk,
            Hq, Hkv, D, (C.c_int64 * 8)(*strides), 1 if causal else 0, float(scale), ws.data_ptr(),
            ws.numel())
    return out, lse


def flash_attn_varlen_bwd(q, k, v, o, do, lse, cu_seqlens, cu_seqlens_kv=None, causal: bool = True,
                          scale: float = 0.0, dq=None, dk=None, dv=None, workspace=None):
    """Backward of flash_attn_varlen_fwd: returns (dQ, dK, dV) shaped like q, k, v, from its
    inputs, its o and lse and the upstream gradient do.  A kv head's dK and dV sum over the query
    heads that share it; the same inputs give the same bits.  dq, dk, dv may be given (parts of a
    fused projection's gradient, for example); rows of no sequence are not written."""
    cu_kv, T, Tk, Hq, Hkv, D = _varlen_shapes(q, k, v, cu_seqlens, cu_seqlens_kv)
    dev, strides = q.device, []
    dq = torch.empty(T, Hq, D, dtype=q.dtype, device=dev) if dq is None else dq
    dk = torch.empty(Tk, Hkv, D, dtype=q.dtype, device=dev) if dk is None else dk
    dv = torch.empty(Tk, Hkv, D, dtype=q.dtype, device=dev) if dv is None else dv
    ptr = [_packed(t, name, n, h, D, dev, strides) for t, name, n, h in (
        (q, "q", T, Hq), (k, "k", Tk, Hkv), (v, "v", Tk, Hkv), (o, "o", T, Hq), (do, "do", T, Hq),
        (dq, "dq", T, Hq), (dk, "dk", Tk, Hkv), (dv, "dv", Tk, Hkv))]
    _check_varlen_lse(lse, Hq, T, dev)
    B = cu_seqlens.numel() - 1
    ws = _workspace(workspace, lib().amp_flash_attn_varlen_bwd_workspace_bytes(B, Hq, T), dev)
    call_on(dev, "amp_flash_attn_varlen_bwd_bf16_dev", *ptr[:5], lse.data_ptr(), *ptr[5:],
            _offsets(cu_seqlens, "cu_seqlens", dev), _offsets(cu_kv, "cu_seqlens_kv", dev), B, T, Tk,
            Hq, Hkv, D, (C.c_int64 * 16)(*strides), 1 if causal else 0, float(scale), ws.data_ptr(),
            ws.numel())
    return dq, dk, dv
