"""Refusals of the rotary positions and the paged cache's append: before any CUDA work."""
import ctypes as C

import pytest
import torch

from amp_b200 import paged, rope
from amp_b200._lib import AmpError, call

P = 1 << 20   # an aligned address that is never read: every call below is refused


def rope_call(q=P, qo=P, k=P, ko=P, dtype=1, T=4, Hq=4, Hk=2, D=64,
              strides=(256, 64, 256, 64, 128, 64, 128, 64), pos=P, stride=4, axes=1, sections=(32,),
              f=P):
    call("amp_rope_dev", q, qo, k, ko, dtype, T, Hq, Hk, D,
         (C.c_int64 * 8)(*strides) if strides else None, pos, stride, axes,
         (C.c_int32 * len(sections))(*sections) if sections else None, f, 0, 0, None)


def append_call(q=P, qo=P, k=P, v=P, T=4, Hq=4, Hkv=2, D=64,
                strides=(256, 64, 256, 64, 128, 64, 128, 64), pos=P, stride=4, axes=1,
                sections=(32,), f=P, kp=P, vp=P, bt=P, ctx=P, cu=P, B=2, pages=9, width=3):
    call("amp_paged_rope_append_bf16_dev", q, qo, k, v, T, Hq, Hkv, D,
         (C.c_int64 * 8)(*strides) if strides else None, pos, stride, axes,
         (C.c_int32 * len(sections))(*sections) if sections else None, f, 0, kp, vp, bt, ctx, cu, B,
         pages, width, None)


SHARED = [(dict(T=-1), -1), (dict(Hq=-1), -1), (dict(D=0), -1), (dict(D=63), -2), (dict(D=2048), -2),
          (dict(strides=None), -1), (dict(axes=5), -2), (dict(axes=-1), -2), (dict(pos=None), -1),
          (dict(f=None), -1), (dict(sections=None), -1), (dict(sections=(-1,)), -1),
          (dict(sections=(33,)), -1), (dict(sections=(16, 16), axes=2, stride=3), -1),
          (dict(q=None), -1), (dict(qo=None), -1), (dict(k=None), -1), (dict(Hq=5000), -2),
          (dict(strides=(0, 64, 256, 64, 128, 64, 128, 64)), -1),
          (dict(strides=(256, 64, 256, -64, 128, 64, 128, 64)), -1),
          (dict(strides=(256, 64, 512, 64, 128, 64, 128, 64)), -1)]


@pytest.mark.parametrize("kw,code", SHARED + [(dict(dtype=2), -2), (dict(ko=None), -1)], ids=str)
def test_rope_refuses(kw, code, amp_lib):
    with pytest.raises(AmpError) as e:
        rope_call(**kw)
    assert e.value.code == code


@pytest.mark.parametrize("kw,code", SHARED + [(dict(B=0), -1), (dict(Hkv=0), -1), (dict(pages=0), -1),
                                              (dict(width=0), -1), (dict(kp=None), -1),
                                              (dict(vp=None), -1), (dict(bt=None), -1),
                                              (dict(ctx=None), -1), (dict(cu=None), -1),
                                              (dict(v=None), -1)], ids=str)
def test_append_refuses(kw, code, amp_lib):
    with pytest.raises(AmpError) as e:
        append_call(**kw)
    assert e.value.code == code


def test_no_tokens_is_no_work(amp_lib):
    rope_call(T=0, q=None)
    rope_call(Hq=0, Hk=0)
    append_call(T=0, k=None)


def test_python_refuses(amp_lib):
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pos, f = torch.zeros(1, 4, dtype=torch.int32), torch.ones(32)
    with pytest.raises(ValueError):
        rope.rope_fwd(q, None, pos, f)        # not on a GPU
    with pytest.raises(ValueError):
        paged.rope_append(q, q, q, q, q, q, q, q, pos, f)


@pytest.mark.parametrize("call_of", [rope_call, append_call])
def test_an_empty_tensor_has_no_address(call_of, amp_lib):
    """What a caller holds for no tokens: positions, q, k and v at address 0; for no pairs, inv_freq too."""
    none = dict(T=0, q=None, k=None, qo=None, pos=None)
    call_of(**none)
    call_of(**none, sections=(0,), f=None)
    call_of(**none, sections=(16, 16), axes=2, stride=0)
    with pytest.raises(AmpError):
        call_of(**none, f=None)       # pairs without frequencies are refused, however many tokens
    with pytest.raises(AmpError):
        call_of(**none, sections=None)


def test_refuses_an_output_in_another_tensors_place(amp_lib):
    q, qo, k, ko = (P + (i << 12) for i in range(4))
    for kw in (dict(qo=k), dict(ko=q), dict(qo=ko), dict(qo=q, ko=q)):
        with pytest.raises(AmpError, match="shares memory") as e:
            rope_call(**(dict(q=q, qo=qo, k=k, ko=ko) | kw))
        assert e.value.code == -1
    for kw in (dict(qo=k), dict(qo=ko)):
        with pytest.raises(AmpError, match="shares memory") as e:
            append_call(**(dict(q=q, qo=qo, k=k, v=ko) | kw))
        assert e.value.code == -1
