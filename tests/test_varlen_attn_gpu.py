"""Packed-sequence attention (forward and backward) on the B200 vs fp64, element by element.

The bounds count roundings (u = 2^-8, half a bf16 step relative to the value):
  O     rounded once, from P rounded once:          u |O| + u P|V|
  lse   fp32 sums of D products:                    D 2^-23 max scale |q|.|k| + a few 2^-22
  dV    rounded once, from P rounded once:          u |dV| + u P^T|dO|
  dS    rounded once, Delta from the bf16 O:        u |dS| + P dDelta,
        dDelta = sum |dO| (u |O| + u P|V|)
  dQ    u |dQ| + scale |err dS| |K|;  dK  u |dK| + scale |err dS|^T |Q|
each with 5% for products of roundings and 1e-5 for the fp32 sums.  The scores' fp32 error
enters P through exp: it is the lse bound, and is added to u wherever P is.
"""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from amp_b200 import attention
from amp_b200._lib import lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
ROOT = Path(__file__).resolve().parents[1]


def make(lens_q, lens_kv, Hq, Hkv, D, seed=0, pad_q=0, pad_kv=0):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(lens_q) + pad_q, sum(lens_kv) + pad_kv
    q, do = (torch.randn(tq, Hq, D, generator=g).to(torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(tk, Hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    cu = [torch.tensor(np.concatenate([[0], np.cumsum(x)]), dtype=torch.int32) for x in (lens_q, lens_kv)]
    return q, k, v, do, *cu


def reference(q, k, v, do, lens_q, lens_kv, causal, scale=0.0):
    """fp64 results and bounds: {name: (value, bound)} for o, lse, dq, dk, dv."""
    q, k, v, do = (x.double().numpy() for x in (q, k, v, do))
    Hq, Hkv, D = q.shape[1], k.shape[1], q.shape[2]
    G, sc = Hq // Hkv, scale if scale > 0 else 1 / np.sqrt(D)
    val = {n: np.zeros(x.shape) for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    err = {n: np.zeros(x.shape) for n, x in val.items()}
    val["lse"], err["lse"] = np.full((Hq, q.shape[0]), -np.inf), np.zeros((Hq, q.shape[0]))
    a = b = 0
    for lq, lk in zip(lens_q, lens_kv):
        Q, K = slice(a, a + lq), slice(b, b + lk)
        a, b = a + lq, b + lk
        if lq == 0 or lk == 0:
            continue
        seen = np.tril(np.ones((lq, lk), bool), lk - lq) if causal else np.ones((lq, lk), bool)
        for h in range(Hq):
            qh, kh, vh, doh = q[Q, h], k[K, h // G], v[K, h // G], do[Q, h]
            s = np.where(seen, sc * (qh @ kh.T), -np.inf)
            e_s = D * 2.0 ** -23 * sc * (np.abs(qh) @ np.abs(kh).T).max() + 4 * 2.0 ** -22
            m = s.max(1, keepdims=True)
            m = np.where(np.isfinite(m), m, 0)
            p = np.exp(s - m)
            l = p.sum(1, keepdims=True)
            with np.errstate(divide="ignore"):
                val["lse"][h, Q] = (m + np.log(l))[:, 0]
            p = p / np.where(l > 0, l, 1)
            err["lse"][h, Q] = e_s + np.where(l[:, 0] > 0, np.abs(m[:, 0]) * 2.0 ** -22, 0)
            u = U + 2 * e_s
            o, o_abs = p @ vh, p @ np.abs(vh)
            val["o"][Q, h] = o
            e_o = err["o"][Q, h] = U * np.abs(o) + u * o_abs
            val["dv"][K, h // G] += p.T @ doh
            err["dv"][K, h // G] += u * (p.T @ np.abs(doh))
            dp = doh @ vh.T
            ds = p * (dp - (doh * o).sum(1, keepdims=True))
            e_ds = u * np.abs(ds) + p * ((np.abs(doh) * e_o).sum(1, keepdims=True)
                                               + D * 2.0 ** -23 * (np.abs(doh) @ np.abs(vh).T))
            val["dq"][Q, h] = sc * (ds @ kh)
            err["dq"][Q, h] = sc * (e_ds @ np.abs(kh))
            val["dk"][K, h // G] += sc * (ds.T @ qh)
            err["dk"][K, h // G] += sc * (e_ds.T @ np.abs(qh))
    for n in ("dq", "dk", "dv"):
        err[n] += U * np.abs(val[n])
    return {n: (val[n], 1.05 * err[n] + 1e-5) for n in val}


def check(got, ref, names):
    for n in names:
        x, (want, bound) = got[n].double().cpu().numpy(), ref[n]
        x = x[:want.shape[0]] if n != "lse" else x[:, :want.shape[1]]
        fin = np.isfinite(want)
        assert np.array_equal(np.isfinite(x), fin), n
        assert np.array_equal(x[~fin], want[~fin]), n
        over = np.abs(x[fin] - want[fin]) / bound[fin]
        assert over.size == 0 or over.max() <= 1, (n, float(over.max()))


def run(q, k, v, do, cu_q, cu_kv, causal, **kw):
    q, k, v, do, cu_q, cu_kv = (x.cuda() for x in (q, k, v, do, cu_q, cu_kv))
    o, lse = attention.flash_attn_varlen_fwd(q, k, v, cu_q, cu_kv, causal=causal, **kw)
    dq, dk, dv = attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu_q, cu_kv, causal=causal, **kw)
    torch.cuda.synchronize()
    assert lib().amp_device_status(1) == 0
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


ALL = ("o", "lse", "dq", "dk", "dv")
SAME = [[1], [128], [129], [17, 0, 1, 127, 300], [256, 5, 0, 0, 640]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (8, 2, 128), (6, 2, 64), (5, 1, 128), (8, 1, 64)])
@pytest.mark.parametrize("lens", SAME, ids=str)
def test_self_attention_lengths(lens, Hq, Hkv, D, causal, cuda, amp_lib):
    q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=len(lens) + Hq)
    check(run(q, k, v, do, cu, cu, causal), reference(q, k, v, do, lens, lens, causal), ALL)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("pairs", [
    [(5, 300), (300, 5), (0, 10), (10, 0), (130, 131)],   # rows and whole sequences that see nothing
    [(1, 1000), (1, 1), (0, 0), (200, 129)],
    [(3, 0), (130, 0)],                                   # no key anywhere
], ids=str)
def test_query_and_key_lengths_differ(pairs, Hq, Hkv, D, causal, cuda, amp_lib):
    lq, lk = zip(*pairs)
    q, k, v, do, cu_q, cu_kv = make(lq, lk, Hq, Hkv, D, seed=7)
    check(run(q, k, v, do, cu_q, cu_kv, causal), reference(q, k, v, do, lq, lk, causal), ALL)


def test_keys_without_any_query_get_zero_gradients(cuda, amp_lib):
    q, k, v, do, cu_q, cu_kv = make([0, 0], [5, 140], 4, 2, 128)
    got = run(q, k, v, do, cu_q, cu_kv, True)
    assert got["o"].shape[0] == 0 and not got["dk"].any() and not got["dv"].any()


@pytest.mark.parametrize("scale", [0.02, 0.5])
def test_scale(scale, cuda, amp_lib):
    lens = [100, 200]
    q, k, v, do, cu, _ = make(lens, lens, 4, 2, 64, seed=3)
    check(run(q, k, v, do, cu, cu, True, scale=scale),
          reference(q, k, v, do, lens, lens, True, scale), ALL)


@pytest.mark.parametrize("Hq,Hkv,lens", [(8, 1, [300, 1, 0, 129]), (7, 1, [1500]), (12, 4, [900, 70]), (28, 4, [513] * 3)])
def test_groups_summed_in_parts(Hq, Hkv, lens, cuda, amp_lib):
    """Few key tiles: the group's query heads are shared out, in parts that need not be equal."""
    for D in (64, 128):
        q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=Hq)
        assert lib().amp_flash_attn_varlen_bwd_workspace_bytes(len(lens), Hq, Hkv, sum(lens), sum(lens), D) \
            > 64 + 1000 + (Hq + 2 * 2 * Hkv * D) * sum(lens) * 4
        check(run(q, k, v, do, cu, cu, True), reference(q, k, v, do, lens, lens, True), ALL)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("pairs", [[(1, 4000)], [(5, 3000), (200, 2500), (0, 700)], [(257, 1100)],
                                   [(40, 5000), (1, 0), (300, 10)]], ids=str)
def test_keys_shared_out_where_queries_are_few(pairs, Hq, Hkv, D, causal, cuda, amp_lib):
    lq, lk = zip(*pairs)
    assert lib().amp_flash_attn_varlen_workspace_bytes(len(lq), Hq, Hkv, sum(lq), sum(lk), D) > sum(lq) * Hq * D * 8
    q, k, v, do, cu_q, cu_kv = make(lq, lk, Hq, Hkv, D, seed=41, pad_q=30, pad_kv=30)
    n, m = sum(lq), sum(lk)
    want = reference(q[:n], k[:m], v[:m], do[:n], lq, lk, causal)
    for x, y in ((q, n), (k, m), (v, m), (do, n)):
        x[y:] = float("nan")
    check(run(q, k, v, do, cu_q, cu_kv, causal), want, ALL)


def test_shared_out_keys_repeat_and_replay(cuda, amp_lib):
    q, k, v, do, cu_q, cu_kv = (x.cuda() for x in make([3, 200], [3000, 2000], 8, 2, 128, seed=43))
    one = attention.flash_attn_varlen_fwd(q, k, v, cu_q, cu_kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two = attention.flash_attn_varlen_fwd(q, k, v, cu_q, cu_kv)
    two[0].fill_(7.0)
    for _ in range(3):
        graph.replay()
        three = attention.flash_attn_varlen_fwd(q, k, v, cu_q, cu_kv)
        for a, b, c in zip(one, two, three):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_more_sequences_than_the_plan_has_threads(cuda, amp_lib):
    lens = [int(n) for n in np.random.default_rng(5).integers(0, 4, 2100)]
    q, k, v, do, cu, _ = make(lens, lens, 2, 1, 64, seed=5)
    check(run(q, k, v, do, cu, cu, True), reference(q, k, v, do, lens, lens, True), ALL)


def test_parts_of_a_fused_projection_and_strided_gradients(cuda, amp_lib):
    lens, Hq, Hkv, D = [70, 200, 1], 8, 2, 128
    q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=9)
    ref = reference(q, k, v, do, lens, lens, True)
    qkv = torch.cat([q, k, v], 1).cuda()
    parts = qkv.split([Hq, Hkv, Hkv], 1)
    o = torch.full((Hq, 271, D), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)   # head major
    grad = torch.full_like(qkv, 7.0)
    dq, dk, dv = grad.split([Hq, Hkv, Hkv], 1)
    _, lse = attention.flash_attn_varlen_fwd(*parts, cu.cuda(), out=o)
    attention.flash_attn_varlen_bwd(*parts, o, do.cuda(), lse, cu.cuda(), dq=dq, dk=dk, dv=dv)
    check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref, ALL)


def test_rows_of_no_sequence_are_not_read_nor_written(cuda, amp_lib):
    lens, Hq, Hkv, D = [60, 130], 4, 2, 128
    for bad in (float("nan"), float("inf")):
        q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=11, pad_q=100, pad_kv=100)
        n = sum(lens)
        ref = reference(q[:n], k[:n], v[:n], do[:n], lens, lens, True)
        for x in (q, k, v, do):
            x[n:] = bad
        qc, kc, vc, doc, cuc = (x.cuda() for x in (q, k, v, do, cu))
        o, dq = (torch.full_like(qc, 7.0) for _ in range(2))
        dk, dv = (torch.full_like(kc, 7.0) for _ in range(2))
        lse = torch.full((Hq, n + 100), 7.0, device="cuda")
        attention.flash_attn_varlen_fwd(qc, kc, vc, cuc, out=o, lse=lse)
        attention.flash_attn_varlen_bwd(qc, kc, vc, o, doc, lse, cuc, dq=dq, dk=dk, dv=dv)
        for x in (o, dq, dk, dv):
            assert (x[n:] == 7.0).all()
        assert (lse[:, n:] == 7.0).all()
        check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref, ALL)


@pytest.mark.parametrize("pairs,Hq,Hkv", [([(60, 60), (130, 130)], 4, 2), ([(5, 3000)], 8, 1)], ids=str)
def test_rows_before_the_first_sequence_are_left_alone(pairs, Hq, Hkv, cuda, amp_lib):
    lq, lk = zip(*pairs)
    q, k, v, do, cu_q, cu_kv = make(lq, lk, Hq, Hkv, 64, seed=12, pad_q=9, pad_kv=13)
    ref = reference(q[9:], k[13:], v[13:], do[9:], lq, lk, True)
    for x, n in ((q, 9), (do, 9), (k, 13), (v, 13)):
        x[:n] = float("nan")
    q, k, v, do, cu_q, cu_kv = (x.cuda() for x in (q, k, v, do, cu_q + 9, cu_kv + 13))
    o, dq = (torch.full_like(q, 7.0) for _ in range(2))
    dk, dv = (torch.full_like(k, 7.0) for _ in range(2))
    lse = torch.full((Hq, len(q)), 7.0, device="cuda")
    attention.flash_attn_varlen_fwd(q, k, v, cu_q, cu_kv, out=o, lse=lse)
    attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu_q, cu_kv, dq=dq, dk=dk, dv=dv)
    assert (lse[:, :9] == 7.0).all() and all((x[:n] == 7.0).all() for x, n in ((o, 9), (dq, 9), (dk, 13), (dv, 13)))
    check({"o": o[9:], "lse": lse[:, 9:], "dq": dq[9:], "dk": dk[13:], "dv": dv[13:]}, ref, ALL)


def test_a_sequence_of_nan_leaves_its_neighbours_alone(cuda, amp_lib):
    lens, Hq, Hkv, D = [60, 33, 200, 7], 4, 2, 64
    q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=13)
    clean = run(q, k, v, do, cu, cu, True)
    bad = slice(60, 93)
    for x in (q, k, v, do):
        x[bad] = float("nan")
    got = run(q, k, v, do, cu, cu, True)
    keep = torch.ones(300, dtype=torch.bool)
    keep[bad] = False
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
    assert torch.equal(got["lse"][:, keep], clean["lse"][:, keep])


def test_gradients_agree_with_differences(cuda, amp_lib):
    """d/de of sum(dO * O(x + e w)) at e = 0 equals sum(grad * w), in fp64 on the oracle's
    formula for the loss and the kernel's gradients: the bf16 gradients are off by at most
    their bound, weighted with |w|."""
    lens = [33, 150]
    q, k, v, do, cu, _ = make(lens, lens, 4, 2, 64, seed=17)
    got = run(q, k, v, do, cu, cu, True)
    ref = reference(q, k, v, do, lens, lens, True)
    g = torch.Generator().manual_seed(1)

    def loss(x):
        return (do.double().numpy() * reference(*x, do, lens, lens, True)["o"][0]).sum()

    for i, n in enumerate(("dq", "dk", "dv")):
        w = torch.randn(ref[n][0].shape, generator=g, dtype=torch.float64)
        e, x = 1e-4, [t.double() for t in (q, k, v)]
        ahead, back = list(x), list(x)
        ahead[i], back[i] = x[i] + e * w, x[i] - e * w
        slope = (loss(ahead) - loss(back)) / (2 * e)
        mine = (got[n].double().cpu() * w).sum().item()
        assert abs(mine - slope) <= (ref[n][1] * w.abs().numpy()).sum() + 1e-6 * abs(slope)


def test_matches_the_rectangular_kernels(cuda, amp_lib):
    B, S, Hq, Hkv, D = 3, 384, 4, 4, 128    # (a group's dK and dV may be summed in parts)
    q, k, v, do, cu, _ = make([S] * B, [S] * B, Hq, Hkv, D, seed=19)
    got = run(q, k, v, do, cu, cu, True)
    dense = [x.cuda().view(B, S, -1, D).transpose(1, 2).contiguous() for x in (q, k, v, do)]
    o, lse = attention.flash_attn_fwd(*dense[:3], True)
    assert torch.equal(got["lse"], lse.transpose(0, 1).reshape(Hq, B * S))
    assert torch.equal(got["o"].view(B, S, Hq, D).transpose(1, 2), o)
    dv = attention.flash_attn_bwd(*dense[:3], o, dense[3], lse, True)[2]
    assert torch.equal(got["dv"].view(B, S, -1, D).transpose(1, 2), dv)


def test_same_bits_again_on_another_stream_and_from_a_graph(cuda, amp_lib):
    lens = [300, 5, 0, 129, 700]
    q, k, v, do, cu, _ = (x.cuda() for x in make(lens, lens, 8, 2, 128, seed=23))
    do = do.contiguous()

    def step():
        o, lse = attention.flash_attn_varlen_fwd(q, k, v, cu)
        return (o, lse, *attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu))

    first = step()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        second = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for x in third:
        x.fill_(7.0)
    # the graph reads the lengths when it runs: other lengths, then the first ones again
    cu2 = cu.clone()
    cu.copy_(torch.tensor([0, 10, 10, 500, 600, 1134], dtype=torch.int32))
    graph.replay()
    expect = step()
    for a, b in zip(third, expect):
        assert torch.equal(a, b)
    cu.copy_(cu2)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert lib().amp_device_status(1) == 0


def test_two_calls_at_once_on_two_streams(cuda, amp_lib):
    jobs = []
    for i in range(2):
        lens = [500, 20, 900] if i else [40, 1200]
        jobs.append([x.cuda() for x in make(lens, lens, 8, 4, 128, seed=29 + i)])
    alone = [attention.flash_attn_varlen_fwd(q, k, v, cu) for q, k, v, _, cu, _ in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    out = [[] for _ in jobs]
    for _ in range(5):
        for i, (q, k, v, _, cu, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                out[i].append(attention.flash_attn_varlen_fwd(q, k, v, cu))
    torch.cuda.synchronize()
    for a, many in zip(alone, out):
        for b in many:
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("offsets", [[0, 50, 40, 100], [0, -3, 100, 100], [0, 50, 100, 101]], ids=str)
def test_offsets_outside_the_tensors_are_skipped_and_reported(offsets, cuda, amp_lib):
    q, k, v, do, _, _ = make([100], [100], 2, 2, 64, seed=31)
    qc, kc, vc = (x.cuda() for x in (q, k, v))
    cu = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = torch.full_like(qc, 7.0)
    attention.flash_attn_varlen_fwd(qc, kc, vc, cu, out=out)
    torch.cuda.synchronize()
    assert lib().amp_device_status(1) == -1 and lib().amp_device_status(1) == 0
    good = [(a, b) for a, b in zip(offsets, offsets[1:]) if 0 <= a <= b <= 100]
    first = good[0]
    if first == (0, 50):
        n = [50]
        # rows that a later sequence names again are that sequence's
        rows = slice(0, 40)
        ref = reference(q[:50], k[:50], v[:50], do[:50], n, n, True)["o"]
        x = out[rows].double().cpu().numpy()
        assert (np.abs(x - ref[0][rows]) <= ref[1][rows]).all()


def test_offsets_past_32_bits(cuda, amp_lib):
    """Tokens 2^30 elements apart, all tensors side by side in one allocation."""
    Hq, Hkv, D, T = 4, 2, 64, 6
    lens = [4, 2]
    far = torch.zeros((T - 1 << 30) + 8192, dtype=torch.bfloat16, device="cuda")
    at = 0

    def view(heads, x=None):
        nonlocal at
        v = far.as_strided((T, heads, D), (1 << 30, D, 1), at)
        at += heads * D
        return v.copy_(x) if x is not None else v

    q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=47)
    ref = reference(q, k, v, do, lens, lens, True)
    qv, kv, vv, dov, o = view(Hq, q), view(Hkv, k), view(Hkv, v), view(Hq, do), view(Hq)
    grads = view(Hq), view(Hkv), view(Hkv)
    _, lse = attention.flash_attn_varlen_fwd(qv, kv, vv, cu.cuda(), out=o)
    attention.flash_attn_varlen_bwd(qv, kv, vv, o, dov, lse, cu.cuda(), dq=grads[0], dk=grads[1], dv=grads[2])
    check(dict(zip(ALL, (o, lse, *grads))), ref, ALL)


FIRST_IN_CAPTURE = """
import torch
from amp_b200 import attention, rope
q, k = torch.randn(64, 4, 64, device="cuda").bfloat16(), torch.randn(64, 2, 64, device="cuda").bfloat16()
cu = torch.tensor([0, 20, 64], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    o, lse = attention.flash_attn_varlen_fwd(q, k, k, cu)
    grads = attention.flash_attn_varlen_bwd(q, k, k, o, q, lse, cu)
graph.replay()
torch.cuda.synchronize()
o2, lse2 = attention.flash_attn_varlen_fwd(q, k, k, cu)
assert torch.equal(o, o2) and torch.equal(lse, lse2)
for a, b in zip(grads, attention.flash_attn_varlen_bwd(q, k, k, o2, q, lse2, cu)):
    assert torch.equal(a, b)
"""


def test_the_first_call_of_a_process_may_be_captured(cuda, amp_lib):
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr


def test_no_key_anywhere_with_many_items(cuda, amp_lib):
    """The dQ pass alone, its items drawn from the counter."""
    lens = [700] * 20
    q, k, v, do, cu, _ = make(lens, lens, 16, 2, 64, seed=37)
    none = torch.zeros(21, dtype=torch.int32)
    for _ in range(5):
        got = run(q, k[:0], v[:0], do, cu, none, True)
        assert not got["dq"].any() and not got["o"].any() and (got["lse"] == -np.inf).all()


@pytest.mark.parametrize("Hq,Hkv,cu_q,cu_kv,Tk", [
    (4, 2, [0, 200, 50, 100], [0, 3000, 500, 2000], 2600),     # keys and heads shared out
    (8, 1, [0, 200, 50, 100], [0, 200, 50, 100], 100),         # heads shared out in the backward
    (8, 1, [0, 200, 50, 100], [0, 3000, 500, 2000], 2600),
    (8, 1, [70, 20, 101, 50, 60], [1900, 100, 4001, 300, 800], 4000),
], ids=str)
def test_a_sequence_after_bad_offsets_is_whole(Hq, Hkv, cu_q, cu_kv, Tk, cuda, amp_lib):
    """Offsets that do not ascend: the last sequence is the only one within its tensors."""
    T, D, B = 100, 64, len(cu_q) - 1
    assert (amp_lib.amp_flash_attn_varlen_workspace_bytes(B, Hq, Hkv, T, Tk, D) > T * Hq * D * 8) == (Tk > 100)
    assert amp_lib.amp_flash_attn_varlen_bwd_workspace_bytes(B, Hq, Hkv, T, Tk, D) \
        > 64 + 1000 + (Hq * T + 2 * Hkv * D * Tk) * 4
    q, k, v, do, _, _ = make([T], [Tk], Hq, Hkv, D, seed=53)
    Q, K = slice(*cu_q[-2:]), slice(*cu_kv[-2:])
    lq, lk = Q.stop - Q.start, K.stop - K.start
    ref = reference(q[Q], k[K], v[K], do[Q], [lq], [lk], True)
    q, k, v, do = (x.cuda() for x in (q, k, v, do))
    cu, cukv = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu_q, cu_kv))
    o, dq = (torch.full_like(q, 7.0) for _ in range(2))
    dk, dv = (torch.full_like(k, 7.0) for _ in range(2))
    lse = torch.full((Hq, T), 7.0, device="cuda")
    attention.flash_attn_varlen_fwd(q, k, v, cu, cukv, out=o, lse=lse)
    attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu, cukv, dq=dq, dk=dk, dv=dv)
    assert amp_lib.amp_device_status(1) == -1 and amp_lib.amp_device_status(1) == 0
    check({"o": o[Q], "lse": lse[:, Q], "dq": dq[Q], "dk": dk[K], "dv": dv[K]}, ref, ALL)
    for x, rows in ((o, Q), (dq, Q), (dk, K), (dv, K), (lse.T, Q)):
        x[rows] = 7.0
        assert (x == 7.0).all()                                # nothing else was written


@pytest.mark.parametrize("times", [16, 51])
def test_overlapping_sequences_get_no_work(times, cuda, amp_lib):
    """The same rows again and again (up to 32 sequences, and more): more tiles than the tensors have."""
    T, Hq, Hkv, D = 1000, 2, 2, 64
    q, k, v, do, _, _ = (x.cuda() for x in make([T], [T], Hq, Hkv, D, seed=59))
    cu = torch.tensor([0, T] * times, dtype=torch.int32, device="cuda")
    o, dq = (torch.full_like(q, 7.0) for _ in range(2))
    dk, dv = (torch.full_like(k, 7.0) for _ in range(2))
    lse = torch.full((Hq, T), 7.0, device="cuda")
    attention.flash_attn_varlen_fwd(q, k, v, cu, out=o, lse=lse)
    assert amp_lib.amp_device_status(1) == -1 and amp_lib.amp_device_status(1) == 0
    attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu, dq=dq, dk=dk, dv=dv)
    assert amp_lib.amp_device_status(1) == -1 and amp_lib.amp_device_status(1) == 0
    assert all((x == 7.0).all() for x in (o, lse, dq, dk, dv))


def test_overlapping_sequences_of_more_items_than_32_bits_count(cuda, amp_lib):
    T, Hq, Hkv, D, B = 8192, 64, 1, 64, 1 << 22        # 2^21 times 2048 items
    q, k, v, _, _, _ = (x.cuda() for x in make([T], [T], Hq, Hkv, D, seed=61))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda").repeat(B // 2 + 1)[:B + 1]
    o, lse = torch.full_like(q, 7.0), torch.full((Hq, T), 7.0, device="cuda")
    attention.flash_attn_varlen_fwd(q, k, v, cu, out=o, lse=lse)
    assert amp_lib.amp_device_status(1) == -1 and amp_lib.amp_device_status(1) == 0
    assert (o == 7.0).all() and (lse == 7.0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("lq,lk,Hq,Hkv,D", [(40, 40, 4, 2, 128), (300, 300, 3, 3, 64), (5, 3000, 8, 2, 128)])
def test_a_query_that_is_not_finite_has_no_finite_lse(lq, lk, Hq, Hkv, D, bad, cuda, amp_lib):
    """-inf is the lse of a row that sees nothing; this one sees keys.  Every other row keeps its bits."""
    q, k, v, _, cu, cukv = (x.cuda() for x in make([lq], [lk], Hq, Hkv, D, seed=67))
    k[:, :, 0] = k[:, :, 0].abs() + 1                     # a query's inf is in every score as +inf
    want = attention.flash_attn_varlen_fwd(q, k, v, cu, cukv)
    q[3, 1, 0] = bad
    got = attention.flash_attn_varlen_fwd(q, k, v, cu, cukv)
    assert got[0][3, 1].isnan().all() and got[1][1, 3].isnan()
    got[0][3, 1], got[1][1, 3] = want[0][3, 1], want[1][1, 3]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if lq == lk:
        dense = [x.transpose(0, 1)[None].contiguous() for x in (q, k, v)]
        o, lse = attention.flash_attn_fwd(*dense, True)
        assert o[0, 1, 3].isnan().all() and lse[0, 1, 3].isnan() and lse.isnan().sum() == 1


@pytest.mark.parametrize("pairs", [[(300, 300), (7, 7), (0, 0), (129, 129)], [(5, 3000), (60, 2500)],
                                   [(700, 700)] * 40], ids=lambda p: str(p[:3]))
def test_output_in_the_place_of_the_queries(pairs, cuda, amp_lib):
    Hq, Hkv, D = 8, 2, 64
    lq, lk = zip(*pairs)
    q, k, v, _, cu, cukv = (x.cuda() for x in make(lq, lk, Hq, Hkv, D, seed=71, pad_q=9))
    want, lse = attention.flash_attn_varlen_fwd(q, k, v, cu, cukv)
    room = torch.cat([q, q], 1)                             # and as part of a larger tensor
    for place in (q, room[:, :Hq]):
        before = place.clone()
        out, lse2 = attention.flash_attn_varlen_fwd(place, k, v, cu, cukv, out=place)
        n = sum(lq)
        assert out is place and torch.equal(place[:n], want[:n]) and torch.equal(lse2[:, :n], lse[:, :n])
        assert torch.equal(place[n:], before[n:])
    with pytest.raises(RuntimeError, match="shares memory"):
        attention.flash_attn_varlen_fwd(q[:n, :Hkv], k[:n], v[:n], cu, out=k[:n])


@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_many_sequences_shared_out(causal, cuda, amp_lib):
    """More sequences than a warp has lanes (the plan kernel's lists), keys shared out and joined."""
    Hq, Hkv, D = 4, 1, 128
    rng = np.random.default_rng(73)
    lq = [int(x) for x in rng.integers(0, 4, 40)]
    lk = [int(x) for x in rng.integers(800, 1300, 40)]
    lk[3] = lq[5] = lq[6] = lk[39] = 0
    n, m = sum(lq), sum(lk)
    assert amp_lib.amp_flash_attn_varlen_workspace_bytes(40, Hq, Hkv, n + 30, m + 50, D) > 2 * (n + 30) * Hq * D * 4
    q, k, v, do, cu_q, cu_kv = make(lq, lk, Hq, Hkv, D, seed=73, pad_q=30, pad_kv=50)
    want = reference(q[:n], k[:m], v[:m], do[:n], lq, lk, causal)
    for x, y in ((q, n), (k, m), (v, m), (do, n)):
        x[y:] = float("nan")
    got = run(q, k, v, do, cu_q, cu_kv, causal)
    check(got, want, ALL)
    again = run(q, k, v, do, cu_q, cu_kv, causal)
    assert torch.equal(got["o"][:n], again["o"][:n]) and torch.equal(got["lse"][:, :n], again["lse"][:, :n])


@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (7, 1)])
def test_heads_of_many_sequences_summed_in_parts(Hq, Hkv, cuda, amp_lib):
    D = 64
    rng = np.random.default_rng(79)
    lens = [int(x) for x in rng.integers(1, 200, 70)]
    lens[0] = lens[33] = lens[69] = 0
    lens[50] = 700
    n = sum(lens)
    assert amp_lib.amp_flash_attn_varlen_bwd_workspace_bytes(70, Hq, Hkv, n + 20, n + 20, D) \
        > 64 + 70 * 24 + (Hq + 2 * 2 * Hkv * D) * (n + 20) * 4
    q, k, v, do, cu, _ = make(lens, lens, Hq, Hkv, D, seed=79, pad_q=20, pad_kv=20)
    want = reference(q[:n], k[:n], v[:n], do[:n], lens, lens, True)
    for x in (q, k, v, do):
        x[n:] = float("nan")
    got = run(q, k, v, do, cu, cu, True)
    check(got, want, ALL)
    again = run(q, k, v, do, cu, cu, True)
    assert all(torch.equal(got[x][:n], again[x][:n]) for x in ("dq", "dk", "dv"))


def test_a_short_wait_limit_holds_for_steps_not_for_whole_items(cuda, amp_lib):
    """Items of several milliseconds under a limit of one: the roles that wait for whole items go on."""
    q, k, v, do, cu, cukv = (x.cuda() for x in make([130000], [519000], 1, 1, 64, seed=83))

    def step():
        o, lse = attention.flash_attn_varlen_fwd(q, k, v, cu, cukv, causal=False)
        return (o, lse, *attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu, cukv, causal=False))

    want = step()
    torch.cuda.synchronize()
    try:
        assert amp_lib.amp_set_wait_timeout_ns(1_000_000) == 0
        got = step()
        assert amp_lib.amp_device_status(1) == 0, amp_lib.amp_last_error()
    finally:
        amp_lib.amp_set_wait_timeout_ns(0)
    assert all(map(torch.equal, want, got))


def rounded(q, k, v, do, lens_q, lens_kv, causal):
    """dQ and dK in fp64 and with dS and the results rounded to bf16: what rounding them costs."""
    q, k, v, do = (x.double() for x in (q, k, v, do))
    G, sc = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    exact, near = [[torch.zeros_like(x) for x in (q, k)] for _ in range(2)]
    a = b = 0
    for lq, lk in zip(lens_q, lens_kv):
        Q, K = slice(a, a + lq), slice(b, b + lk)
        a, b = a + lq, b + lk
        kk, vv = (x[K].repeat_interleave(G, 1) for x in (k, v))
        s = sc * torch.einsum("ihd,jhd->hij", q[Q], kk)
        if causal:
            s = s.masked_fill(~torch.ones(lq, lk, dtype=torch.bool).tril(lk - lq), -torch.inf)
        p = s.softmax(2).nan_to_num(0.0)
        dp = torch.einsum("ihd,jhd->hij", do[Q], vv)
        ds = p * (dp - (p * dp).sum(2, keepdim=True))
        for out, x in ((exact, ds), (near, ds.bfloat16().double())):
            out[0][Q] = sc * torch.einsum("hij,jhd->ihd", x, kk)
            out[1][K] = sc * torch.einsum("hij,ihd->jhd", x, q[Q]).unflatten(1, (-1, G)).sum(2)
    return exact, [x.bfloat16().double() for x in near]


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 8, 64), (8, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("lens_q,lens_kv,causal", [
    ([3] * 60, [3] * 60, True), ([8] * 50 + [20] * 20, [8] * 50 + [20] * 20, True), ([1, 33, 17, 90, 64, 700, 31], [1, 33, 17, 90, 64, 700, 31], True),
    ([40, 9, 5, 16, 200], [20, 12, 32, 31, 3], True), ([40, 9, 5, 160, 3, 16], [20, 12, 32, 31, 0, 16], False), ([50] * 20, [33] * 20, False),
], ids=["3", "8 and 20", "mixed", "other lengths", "full", "full, 33 keys"])
def test_few_keys_cost_no_precision(lens_q, lens_kv, causal, Hq, Hkv, D, cuda, amp_lib):
    """In a row of few keys Delta from the rounded O moved every dS by up to twice its own rounding.  What
    is left is the rounding of dS and of the results; 10% are for rows of more than 32 keys, whose
    Delta does come from O: there rounding O adds at most 1 / 33 of the variance for each of
    O's and P's rounding, and the errors of dS in a row, which it shares, add up at most threefold."""
    q, k, v, do, cu_q, cu_kv = make(lens_q, lens_kv, Hq, Hkv, D, seed=89)
    got = run(q, k, v, do, cu_q, cu_kv, causal)
    exact, near = rounded(q, k, v, do, lens_q, lens_kv, causal)
    for name, e, n in zip(("dq", "dk"), exact, near):
        mine = (got[name].double().cpu() - e).norm()
        assert mine <= 1.1 * (n - e).norm(), (name, float(mine / (n - e).norm()))
    check(got, reference(q, k, v, do, lens_q, lens_kv, causal), ALL)
    again = run(q, k, v, do, cu_q, cu_kv, causal)
    assert all(torch.equal(got[x], again[x]) for x in ALL)


def test_overlapping_sequences_of_few_keys_get_no_work(cuda, amp_lib):
    """All rows of a sequence of few keys have their Delta formed by themselves: 2^17 times a million
    rows would be hours."""
    T, B = 1 << 20, 1 << 18
    q, k, v, do, _, _ = (x.cuda() for x in make([T], [16], 1, 1, 64, seed=97))
    cu, cukv = (torch.tensor([0, n], dtype=torch.int32, device="cuda").repeat(B // 2) for n in (T, 16))
    o, lse = torch.zeros_like(q), torch.zeros(1, T, device="cuda")
    dq, dk, dv = (torch.full_like(x, 7.0) for x in (q, k, v))
    attention.flash_attn_varlen_bwd(q, k, v, o, do, lse, cu, cukv, causal=False, dq=dq, dk=dk, dv=dv)
    assert amp_lib.amp_device_status(1) == -1 and amp_lib.amp_device_status(1) == 0
    assert all((x == 7.0).all() for x in (dq, dk, dv))
