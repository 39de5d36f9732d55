"""Rotary positions and the paged cache's append on the B200 vs fp64.

Bound of a turned element: half a step of its type (bf16 2^-8, fp32 2^-24, relative) for the one
rounding, and (|x| + |y|) * 2^-20 for the fp32 turn: the reduced angle as a float is off by at
most pi 2^-24, its sine and cosine by 2 ulp (2^-23), the two products and the sum by 2^-23.
What passes through, and the cache's v, is copied: equal bits.
"""
import numpy as np
import pytest
import torch

from amp_b200 import paged, rope
from amp_b200._lib import lib

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def turned(x, pos, inv_freq, sections, inter, back=False):
    """(value, bound) in fp64."""
    x = x.double().cpu()
    axis = np.repeat(np.arange(len(sections)), sections)
    phi = (pos.cpu().double()[axis].T * inv_freq.cpu().double())[:, None]
    c, s = phi.cos(), phi.sin() * (-1 if back else 1)
    n = phi.shape[2]
    out, near = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if inter else (slice(0, n), slice(n, 2 * n))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    near[..., a] = near[..., b] = x[..., a].abs() + x[..., b].abs()
    return out, near


def check(got, want, half):
    value, near = want
    d = (got.double().cpu() - value).abs()
    assert (d <= half * value.abs() * (near > 0) + near * 2.0 ** -20).all(), float(d.max())


def inputs(T, Hq, Hk, D, sections, dtype, seed=0, far=10000):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(T, h, D, generator=g).to(dtype).cuda() for h in (Hq, Hk))
    pos = torch.randint(0, far, (len(sections), T), generator=g, dtype=torch.int32).cuda()
    n = sum(sections)
    inv_freq = (10000.0 ** (-torch.arange(n) / max(n, 1))).float().cuda()
    return q, k, pos, inv_freq


# head dimension, sections: whole heads, heads turned in part, pair counts that divide no vector
SHAPES = [(128, (16, 24, 24)), (64, (32,)), (128, (10, 6)), (80, (20,)), (80, (7, 5, 3)), (96, (24, 12, 12)),
          (256, (40, 40, 40, 8)), (2, (1,)), (6, (2,)), (128, (0, 64))]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,sections", SHAPES, ids=str)
@pytest.mark.parametrize("T,Hq,Hk", [(1, 4, 1), (37, 3, 2), (600, 1, 1), (3000, 8, 2)])
def test_forward_and_backward(T, Hq, Hk, D, sections, dtype, inter, cuda, amp_lib):
    q, k, pos, f = inputs(T, Hq, Hk, D, sections, dtype, seed=T + D)
    for call, back in ((rope.rope_fwd, False), (rope.rope_bwd, True)):
        a, b = call(q, k, pos, f, sections, inter)
        check(a, turned(q, pos, f, sections, inter, back), HALF[dtype])
        check(b, turned(k, pos, f, sections, inter, back), HALF[dtype])


def test_far_and_negative_positions(cuda, amp_lib):
    q, k, pos, f = inputs(64, 2, 2, 128, (64,), torch.float32)
    far = torch.tensor([2 ** 20 - 1, 1 << 24, 2 ** 31 - 1, -5, -(1 << 20), 0], dtype=torch.int32)
    pos[0, :6] = far.cuda()
    a, _ = rope.rope_fwd(q, None, pos, f)
    # the 64-bit product of a position of 2^31 is off by 2^-53 of 2^31 radians: below the bound
    check(a, turned(q, pos, f, (64,), False), HALF[torch.float32])


def test_gradient_is_the_transpose(cuda, amp_lib):
    """<w, R x> = <R' w, x> for the gradient R' of R, and differences of the linear map are exact."""
    x, w, pos, f = inputs(50, 4, 4, 64, (12, 20), torch.float32, seed=3)
    for inter in (False, True):
        rx, _ = rope.rope_fwd(x, None, pos, f, (12, 20), inter)
        gw, _ = rope.rope_bwd(w, None, pos, f, (12, 20), inter)
        a, b = (w.double() * rx.double()).sum(), (gw.double() * x.double()).sum()
        assert abs(a - b) <= 2 * 2.0 ** -20 * (w.abs().double() * x.abs().double()).sum() * 4


def test_strides_in_place_and_one_position_row(cuda, amp_lib):
    T, Hq, Hkv, D = 300, 8, 2, 128
    q, k, pos, f = inputs(T, Hq, Hkv, D, (64,), torch.bfloat16, seed=5)
    want_q, want_k = rope.rope_fwd(q, k, pos[0], f)
    qkv = torch.cat([q, k, k], 1)
    a, b, rest = qkv.split([Hq, Hkv, Hkv], 1)
    got = rope.rope_fwd(a, b, pos, f)
    assert torch.equal(got[0], want_q) and torch.equal(got[1], want_k)
    rope.rope_fwd(a, b, pos, f, out_q=a, out_k=b)
    assert torch.equal(a, want_q) and torch.equal(b, want_k) and torch.equal(rest, k)
    odd = torch.zeros(T * Hq * (D + 3) + 1, dtype=torch.bfloat16, device="cuda")[1:]
    odd = odd.view(T, Hq, D + 3)[..., :D]           # odd strides and an odd address
    rope.rope_fwd(q, None, pos, f, out_q=odd)
    assert torch.equal(odd, want_q)
    head_major = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rope.rope_fwd(head_major, None, pos, f)[0], want_q)


def test_one_row_of_positions_for_every_axis(cuda, amp_lib):
    q, k, pos, f = inputs(40, 4, 2, 128, (64,), torch.bfloat16, seed=6)
    want, got = rope.rope_fwd(q, k, pos, f), rope.rope_fwd(q, k, pos.expand(3, 40), f, (16, 24, 24))
    assert all(map(torch.equal, got, want))


def test_a_tensor_without_storage_is_an_error(cuda, amp_lib):
    """It has a CUDA device, a type and sizes, so only the address is missing."""
    class Bare(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, *args):
            raise NotImplementedError

    q, _, pos, f = inputs(4, 2, 1, 64, (32,), torch.bfloat16)
    bare = torch.Tensor._make_wrapper_subclass(Bare, (4, 2, 64), dtype=q.dtype, device=q.device)
    with pytest.raises(RuntimeError, match="NULL|storage"):
        rope.rope_fwd(bare, None, pos, f)
    assert torch.equal(rope.rope_fwd(q, None, pos, f)[0], rope.rope_fwd(q.clone(), None, pos, f)[0])


def cache(ctx, Hkv, D, seed=0, spare=3):
    rng = np.random.default_rng(seed)
    need = [-(-c // 16) for c in ctx]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(ctx), max(need) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pools = [torch.full((pages, Hkv, 16, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    return pools, torch.from_numpy(table).cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda")


def expected_pools(shape, table, ctx, lens, k, v):
    """Pools of sevens with the new tokens written, (value, near) for k and bits for v."""
    (kv, kn), out = k, [torch.full(shape, 7.0, dtype=torch.float64) for _ in range(2)]
    near, at = torch.zeros(shape, dtype=torch.float64), 0
    for b, n in enumerate(lens):
        for i in range(n):
            t = ctx[b] - n + i
            page = table[b, t // 16]
            out[0][page, :, t % 16], out[1][page, :, t % 16] = kv[at], v[at].double().cpu()
            near[page, :, t % 16] = kn[at]
            at += 1
    return out, near


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,sections", [(128, (16, 24, 24)), (64, (16,)), (80, (20, 0, 7))], ids=str)
@pytest.mark.parametrize("lens,ctx", [
    ([1] * 5, [1, 16, 17, 500, 33]),                   # a decode step
    ([0, 40, 1, 0, 300], [9, 40, 16, 0, 1000]),        # prompts, some behind a cached prefix, some empty
    ([700], [700]),
], ids=str)
def test_append(lens, ctx, D, sections, inter, cuda, amp_lib):
    Hq, Hkv, T = 6, 2, sum(lens)
    q, k, pos, f = inputs(T, Hq, Hkv, D, sections, torch.bfloat16, seed=T)
    v = torch.randn(T, Hkv, D, device="cuda").bfloat16()
    pools, table, ctxd = cache(ctx, Hkv, D, seed=T)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    qkv = torch.cat([q, k, v], 1)
    parts = qkv.split([Hq, Hkv, Hkv], 1)
    out = paged.rope_append(*parts, *pools, table, ctxd, cu, pos, f, sections, inter)
    check(out, turned(q, pos, f, sections, inter), HALF[torch.bfloat16])
    want, near = expected_pools(pools[0].shape, table.cpu(), ctx, lens, turned(k, pos, f, sections, inter), v)
    check(pools[0], (want[0], near), HALF[torch.bfloat16])
    assert torch.equal(pools[1].double().cpu(), want[1])
    fresh, _, _ = cache(ctx, Hkv, D, seed=T)
    paged.append(k, v, *fresh, table, ctxd, cu)
    plain, _ = expected_pools(pools[0].shape, table.cpu(), ctx, lens, (k.double().cpu(), torch.zeros(k.shape)), v)
    assert torch.equal(fresh[0].double().cpu(), plain[0]) and torch.equal(fresh[1].double().cpu(), plain[1])
    assert lib().amp_device_status(1) == 0


def test_append_skips_padding_and_reports_missing_pages(cuda, amp_lib):
    Hq, Hkv, D = 4, 2, 64
    pools, table, ctx = cache([40, 20], Hkv, D)
    q, k, pos, f = inputs(50, Hq, Hkv, D, (32,), torch.bfloat16)
    cu = torch.tensor([3, 33, 43], dtype=torch.int32, device="cuda")   # rows 0-2 and 43-49 are no one's
    out = torch.full_like(q, 7.0)
    paged.rope_append(q, k, k, *pools, table, ctx, cu, pos, f, out_q=out)
    assert lib().amp_device_status(1) == 0
    assert (out[:3] == 7.0).all() and (out[43:] == 7.0).all()
    assert torch.equal(out[3:43], rope.rope_fwd(q, None, pos, f)[0][3:43])
    assert int((pools[1] != 7.0).any(3).sum()) == Hkv * 40
    # a page number outside the pool, a missing page, a context shorter than its new tokens and
    # one longer than its row: nothing is written for those tokens
    for change in (lambda t, c: t[0].fill_(10 ** 6), lambda t, c: t[0].fill_(-1),
                   lambda t, c: c[:1].fill_(-10), lambda t, c: c[:1].fill_(10 ** 6)):
        fresh, t, c = cache([40, 20], Hkv, D)
        change(t, c)
        paged.append(k, k, *fresh, t, c, cu)
        assert lib().amp_device_status(1) == -1 and lib().amp_device_status(1) == 0
        assert int((fresh[1] != 7.0).any(3).sum()) <= Hkv * 10


def test_offsets_out_of_order_stay_inside(cuda, amp_lib):
    pools, table, ctx = cache([40, 20, 30], 2, 64)
    _, k, _, _ = inputs(50, 1, 2, 64, (32,), torch.bfloat16)
    for cu in ([0, 50, 10, 20], [60, 70, 80, 90], [-5, -4, -3, -2]):
        paged.append(k, k, *pools, table, ctx, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    lib().amp_device_status(1)


def test_page_offsets_past_32_bits(cuda, amp_lib):
    Hkv, D = 8, 128
    pages = (1 << 32) // (Hkv * 16 * D) + 64          # the last pages start past 2^32 elements
    pools = [torch.zeros(pages, Hkv, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.tensor([[pages - 1, 0], [pages - 9, -1]], dtype=torch.int32, device="cuda")
    ctx = torch.tensor([16, 5], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    k = torch.randn(3, Hkv, D, device="cuda").bfloat16()
    paged.append(k, k, *pools, table, ctx, cu)
    for pool in pools:
        assert torch.equal(pool[pages - 1, :, 14], k[0]) and torch.equal(pool[pages - 1, :, 15], k[1])
        assert torch.equal(pool[pages - 9, :, 4], k[2])
        assert int((pool[0] != 0).sum()) == 0


def test_graph_and_other_stream(cuda, amp_lib):
    q, k, pos, f = inputs(16, 8, 2, 128, (64,), torch.bfloat16)
    pools, table, ctx = cache([40] * 16, 2, 128)
    cu = torch.arange(17, dtype=torch.int32, device="cuda")
    first = paged.rope_append(q, k, k, *pools, table, ctx, cu, pos, f)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        second = paged.rope_append(q, k, k, *pools, table, ctx, cu, pos, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = paged.rope_append(q, k, k, *pools, table, ctx, cu, pos, f)
    third.fill_(7.0)
    pools[0].fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, second) and torch.equal(first, third)
    assert torch.equal(pools[0][table[0, 2].item(), :, 7], rope.rope_fwd(k, None, pos, f)[0][0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_tokens(dtype, cuda, amp_lib):
    for sections in ((32,), (8, 12, 12)):
        q, k, pos, f = inputs(0, 4, 2, 64, sections, dtype)
        for call in (rope.rope_fwd, rope.rope_bwd):
            a, b = call(q, k, pos, f, sections)
            assert a.shape == q.shape and b.shape == k.shape
            assert call(q, None, pos, f, sections)[0].shape == q.shape
        if dtype == torch.bfloat16:
            pools, table, ctx = cache([5, 17], 2, 64)
            cu = torch.zeros(3, dtype=torch.int32, device="cuda")
            assert paged.rope_append(q, k, k, *pools, table, ctx, cu, pos, f, sections).shape == q.shape
            paged.append(k, k, *pools, table, ctx, cu)
            assert all((p == 7.0).all() for p in pools)
    assert rope.rope_fwd(q, k, pos[0], f)[0].shape == q.shape
    torch.cuda.synchronize()
    assert lib().amp_device_status(1) == 0


def test_no_pairs_is_a_copy(cuda, amp_lib):
    q, k, pos, f = inputs(37, 3, 2, 80, (0,), torch.bfloat16)
    assert f.numel() == 0
    for sections in (None, (0,)):
        a, b = rope.rope_fwd(q, k, pos, f, sections)
        assert torch.equal(a, q) and torch.equal(b, k)
    pools, table, ctx = cache([37], 2, 80)
    cu = torch.tensor([0, 37], dtype=torch.int32, device="cuda")
    assert torch.equal(paged.rope_append(q, k, k, *pools, table, ctx, cu, pos, f), q)
    fresh, _, _ = cache([37], 2, 80)
    paged.append(k, k, *fresh, table, ctx, cu)
    assert all(map(torch.equal, pools, fresh))
