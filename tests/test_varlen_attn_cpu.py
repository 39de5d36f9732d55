"""Refusals of the packed-sequence attention: argument errors return before any CUDA work."""
import ctypes as C

import pytest
import torch

from amp_b200 import attention
from amp_b200._lib import AmpError, call

FWD, BWD = "amp_flash_attn_varlen_fwd_bf16_dev", "amp_flash_attn_varlen_bwd_bf16_dev"
P = 1 << 20   # an aligned address that is never read: every call below is refused


def fwd(q=P, k=P, v=P, o=P, lse=P, cu=P, cu_kv=P, B=2, tq=10, tk=10, Hq=4, Hkv=2, D=64,
        strides=(256, 64, 128, 64, 128, 64, 256, 64), ws=P, ws_bytes=1 << 20):
    call(FWD, q, k, v, o, lse, cu, cu_kv, B, tq, tk, Hq, Hkv, D,
         (C.c_int64 * 8)(*strides) if strides else None, 1, 0.0, ws, ws_bytes, None)


def bwd(q=P, k=P, v=P, o=P, do=P, lse=P, dq=P, dk=P, dv=P, cu=P, cu_kv=P, B=2, tq=10, tk=10, Hq=4,
        Hkv=2, D=64, strides=(256, 64) * 8, ws=P, ws_bytes=1 << 20):
    call(BWD, q, k, v, o, do, lse, dq, dk, dv, cu, cu_kv, B, tq, tk, Hq, Hkv, D,
         (C.c_int64 * 16)(*strides) if strides else None, 1, 0.0, ws, ws_bytes, None)


BAD = [(dict(B=0), -1), (dict(Hq=0), -1), (dict(Hkv=0), -1), (dict(Hq=5), -1), (dict(tq=-1), -1),
       (dict(tk=-1), -1), (dict(D=80), -2), (dict(D=256), -2), (dict(cu=None), -1),
       (dict(cu_kv=None), -1), (dict(strides=None), -1), (dict(ws=None), -1), (dict(ws=P + 8), -1),
       (dict(ws_bytes=16), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(q=P + 2), -1),
       (dict(v=P + 8), -1), (dict(tq=1 << 30, Hq=4), -2), (dict(B=1 << 30), -2)]


@pytest.mark.parametrize("kw,code", BAD, ids=[str(b[0]) for b in BAD])
@pytest.mark.parametrize("entry", [fwd, bwd])
def test_refused_arguments(entry, kw, code, amp_lib):
    if "tq" in kw or "B" in kw:
        kw = dict(kw, ws_bytes=1 << 62)
    with pytest.raises(AmpError) as e:
        entry(**kw)
    assert e.value.code == code


@pytest.mark.parametrize("stride", [0, -64, 4, 65, 1 << 40])
@pytest.mark.parametrize("entry,n", [(fwd, 8), (bwd, 16)])
def test_refused_strides(entry, n, stride, amp_lib):
    for i in range(n):
        s = [256, 64] * (n // 2)
        s[i] = stride
        with pytest.raises(AmpError) as e:
            entry(strides=s)
        assert e.value.code == -1


def test_no_tokens_is_no_work(amp_lib):
    fwd(tq=0, q=None, o=None)
    bwd(tq=0, tk=0, q=None, k=None)


def test_workspace_sizes(amp_lib):
    fwd_bytes = amp_lib.amp_flash_attn_varlen_workspace_bytes
    assert fwd_bytes(0, 8, 8, 100, 100, 64) == 0
    small, large = (fwd_bytes(b, 8, 8, 100, 100, 64) for b in (1, 1000))
    assert 0 < small < large
    # few queries over many keys: O and lse of the splits
    assert fwd_bytes(1, 8, 8, 16, 10000, 64) > small + 2 * 16 * 8 * 65 * 4
    assert fwd_bytes(1, 8, 8, 10 ** 5, 10 ** 5, 64) <= small + 16
    bwd_bytes = amp_lib.amp_flash_attn_varlen_bwd_workspace_bytes
    assert bwd_bytes(1, 8, 8, 100, 100, 64) >= small + 8 * 100 * 4
    # few key tiles and a group of 8: fp32 sums of its parts, of dK and of dV
    assert bwd_bytes(1, 8, 1, 100, 100, 64) >= small + 8 * 100 * 4 + 8 * 2 * 100 * 64 * 4
    assert bwd_bytes(1, 8, 1, 10 ** 6, 10 ** 6, 64) < 64 + 1000 + 8 * 10 ** 6 * 4
    assert bwd_bytes(1, 8, 8, -1, 100, 64) == 0 and bwd_bytes(1, 8, 3, 100, 100, 64) == 0


def test_python_refuses_what_the_kernels_cannot_read(amp_lib):
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        attention.flash_attn_varlen_fwd(q, q, q, cu)          # not on a GPU
    with pytest.raises(ValueError):
        attention.flash_attn_varlen_fwd(q[0], q, q, cu)       # not packed


def test_keys_are_shared_out_only_where_ctas_are_idle(amp_lib):
    """One query tile a sequence: with a group of 1 a kv head is an item of its own, with an odd group
    half of one more than its heads fill."""
    size = amp_lib.amp_flash_attn_varlen_workspace_bytes

    def shared(B, Hq, Hkv, lq=1, lk=4096):
        return size(B, Hq, Hkv, B * lq, B * lk, 128) > size(B, Hq, Hkv, B * lq, B, 128)

    assert shared(4, 64, 8) and shared(1, 64, 64) and shared(2, 64, 64)     # 128, 64, 128 items
    assert not shared(4, 64, 64) and not shared(40, 12, 4)                  # 256, 320
    assert shared(4, 28, 4) and not shared(40, 28, 4)                       # 64, 640


def apart(names, **kw):
    """Addresses of their own for tensors that stay unread."""
    return {n: P + (i << 12) for i, n in enumerate(names)} | kw


FWD_TENSORS, BWD_TENSORS = ("q", "k", "v", "o"), ("q", "k", "v", "o", "do", "dq", "dk", "dv")


@pytest.mark.parametrize("other", ["k", "v"])
def test_forward_refuses_o_in_the_place_of_keys(other, amp_lib):
    at = apart(FWD_TENSORS)
    with pytest.raises(AmpError, match="shares memory") as e:
        fwd(**at | {"o": at[other]})
    assert e.value.code == -1


def test_forward_refuses_o_over_q_at_other_strides(amp_lib):
    at = apart(FWD_TENSORS)
    for strides in ((256, 64, 128, 64, 128, 64, 512, 64), (256, 64, 128, 64, 128, 64, 256, 128)):
        with pytest.raises(AmpError, match="shares memory"):
            fwd(**at | {"o": at["q"]}, strides=strides)


@pytest.mark.parametrize("grad", ["dq", "dk", "dv"])
@pytest.mark.parametrize("other", BWD_TENSORS)
def test_backward_refuses_a_gradient_in_another_tensors_place(grad, other, amp_lib):
    if grad == other:
        return
    at = apart(BWD_TENSORS)
    with pytest.raises(AmpError, match="share") as e:
        bwd(**at | {grad: at[other]})
    assert e.value.code == -1
