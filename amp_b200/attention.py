"""FlashAttention-2: host-side mirror of kernels/flash_attn.cuh, its backward, and
both over packed sequences of different lengths.

``launch_flash_attn_bf16(Q, K, V, O, lse, B, S_q, S_kv, cfg)`` mirrors
``AMP::launch_flash_attn_bf16`` (kernels/flash_attn.cuh:50-58) with the same
AttnCfg fields (flash_attn.cuh:26-36).  The tile fields Br/Bc are accepted for
source compatibility; the sm_100a kernel always uses 128x128 tiles.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._lib import call, lib, ops


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


def flash_attn_varlen_fwd(q, k, v, cu_seqlens, cu_seqlens_kv=None, causal: bool = True,
                          scale: float = 0.0, out=None, lse=None, workspace=None):
    """Attention over packed sequences: returns (O [tokens, Hq, D], lse [Hq, tokens]).

    q [tokens, Hq, D], k and v [kv tokens, Hkv, D]: bf16, any token and head strides that are
    multiples of 8 elements, so that parts of one fused projection are taken as they are.
    Sequence b is rows cu_seqlens[b] .. cu_seqlens[b+1] of q, and of k and v by cu_seqlens_kv
    (int32 CUDA tensors; cu_seqlens when None).  Under the causal mask the last query sees every
    key of its sequence.  A query that sees none gets O = 0 and lse = -inf.  Rows that belong to
    no sequence are not written: in outputs allocated here they are unspecified.  out may be q, and
    shares no memory with k or v.  A workspace (uint8, amp_flash_attn_varlen_workspace_bytes) must
    not be shared by calls that may overlap."""
    return ops().varlen_fwd(q, k, v, cu_seqlens, cu_seqlens_kv, causal, scale, out, lse, workspace)


def flash_attn_varlen_bwd(q, k, v, o, do, lse, cu_seqlens, cu_seqlens_kv=None, causal: bool = True,
                          scale: float = 0.0, dq=None, dk=None, dv=None, workspace=None):
    """Backward of flash_attn_varlen_fwd: returns (dQ, dK, dV) shaped like q, k, v, from its
    inputs, its o and lse and the upstream gradient do.  A kv head's dK and dV sum over the query
    heads that share it; the same inputs give the same bits.  dq, dk, dv may be given (parts of a
    fused projection's gradient, for example) and share no memory with the inputs; rows of no
    sequence are not written."""
    return ops().varlen_bwd(q, k, v, o, do, lse, cu_seqlens, cu_seqlens_kv, causal, scale, dq, dk, dv,
                            workspace)
