"""The packed and paged operators together, as a model uses them: a serving run (extend, rotate and
append, attend, fork, decode, compact, free) and a training step (rotate, attend, both backwards).

Each stage is checked on what the stage before it really produced, with that stage's bounds
(test_varlen_attn_gpu, test_rope_gpu); decode against fp64 over the pages' contents.
"""
import numpy as np
import pytest
import torch

from oracle import attention as ref
from amp_b200 import attention, paged, rope
from amp_b200._lib import lib
from test_rope_gpu import HALF, check as check_turn, turned
from test_varlen_attn_gpu import U, check, reference

pytestmark = pytest.mark.gpu
HQ, HKV, D, SECTIONS = 8, 2, 128, (16, 24, 24)
LAYERS = 2


def freq():
    return (10000.0 ** (-torch.arange(64) / 64)).float().cuda()


def projection(gen, tokens):
    qkv = torch.randn(tokens, HQ + 2 * HKV, D, generator=gen).to(torch.bfloat16).cuda()
    return qkv.split([HQ, HKV, HKV], 1)


class Server:
    def __init__(self, rows, pages, width, seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.k, self.v = (torch.zeros(LAYERS, pages, HKV, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.ctx = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.freq = freq()

    def write(self, lens):
        """New tokens for every row (0: none): pages, then q, k, v of each layer, attention over the
        new tokens' own keys where the row was empty before.  Returns per layer (q', new k', v)."""
        before = self.ctx.cpu().numpy().copy()
        self.ctx, done = paged.extend_sequences(self.k, self.v, self.table, self.ctx, ints(lens))
        assert done.all()
        cu = ints(np.concatenate([[0], np.cumsum(lens)]))
        pos = np.concatenate([b + np.arange(n) for b, n in zip(before, lens)] + [np.zeros(0, int)])
        pos = ints(np.stack([pos, pos // 2, pos % 7]))
        out = []
        for layer in range(LAYERS):
            q, k, v = projection(self.gen, sum(lens))
            qt = paged.rope_append(q, k, v, self.k[layer], self.v[layer], self.table, self.ctx, cu, pos, self.freq, SECTIONS)
            check_turn(qt, turned(q, pos, self.freq, SECTIONS, False), HALF[torch.bfloat16])
            kt = rope.rope_fwd(k, None, pos, self.freq, SECTIONS)[0]
            out.append((qt, kt, v))
        return cu, out

    def decode(self, q, layer):
        return paged.paged_attn_decode(q, self.k[layer], self.v[layer], self.table, self.ctx, int(self.ctx.max()))[0]

    def check_decode(self, q, layer):
        got = self.decode(q, layer).double().cpu().numpy()
        kp, vp = (x[layer].float().cpu().numpy() for x in (self.k, self.v))
        for b, n in enumerate(self.ctx.tolist()):
            if n == 0:
                continue
            k, v = (ref.paged_gather(x, self.table[b].cpu().numpy(), n)[None] for x in (kp, vp))
            qb = q[b].float().cpu().numpy()[None, :, None]
            o, _ = ref.flash_attn_fwd(qb, k, v, causal=False)
            spread, _ = ref.flash_attn_fwd(qb, k, np.abs(v), causal=False)
            # O and P rounded to bf16 once each, 5% for the rest
            assert (np.abs(got[b] - o[0, :, 0]) <= 1.05 * U * (np.abs(o) + spread)[0, :, 0] + 1e-4).all()
        return got


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def test_serving(cuda, amp_lib):
    rows = 6
    s = Server(rows, pages=120, width=40)
    lens = [200, 33, 16, 0, 0, 0]
    cu, layers = s.write(lens)
    for layer, (q, k, v) in enumerate(layers):
        o, lse = attention.flash_attn_varlen_fwd(q, k, v, cu)
        want = reference(q.cpu(), k.cpu(), v.cpu(), q.cpu(), lens, lens, True)
        check({"o": o, "lse": lse}, want, ("o", "lse"))
        # the prompt's last tokens attend the same through their pages: both within the bound
        for b, n in enumerate(lens[:3]):
            end = int(cu[b + 1])
            last = q[end - 16:end].transpose(0, 1)[None].contiguous()
            op, _ = paged.paged_attn_prefill(last, s.k[layer], s.v[layer], s.table[b:b + 1], s.ctx[b:b + 1])
            d = (op[0].transpose(0, 1).double() - o[end - 16:end].double()).abs().cpu().numpy()
            assert (d <= 2 * want["o"][1][end - 16:end]).all()
    # three samples of row 0 and one of row 1
    assert paged.fork_sequences(s.k, s.v, s.table, s.ctx, ints([0, 0, 1]), ints([3, 4, 5])).all()
    assert s.ctx.tolist() == [200, 33, 16, 200, 200, 33]
    for step in range(20):
        cu, layers = s.write([1] * rows)
        for layer, (q, _, _) in enumerate(layers):
            s.check_decode(q, layer)
    # what the samples wrote is theirs alone: 200 shared tokens, 20 of their own
    k = [ref.paged_gather(s.k[0].float().cpu().numpy(), s.table[b].cpu().numpy(), 220) for b in (0, 3, 4)]
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert np.array_equal(k[a][:, :200], k[b][:, :200]) and not np.array_equal(k[a][:, 200:], k[b][:, 200:])
    # two sequences end, the cache is drawn together, and the others decode as before
    q = torch.randn(rows, HQ, D, device="cuda").bfloat16()
    paged.free_sequences(s.table, s.ctx, ints([1, 3]))
    before = [s.check_decode(q, layer) for layer in range(LAYERS)]
    s.table, used = paged.compact_pages(s.k, s.v, s.table, s.ctx)
    assert int(s.table.max()) == used.item() - 1
    for layer in range(LAYERS):
        s.k[layer, used.item():] = float("nan")     # pages given back
        assert np.array_equal(s.check_decode(q, layer), before[layer])
    s.write([1, 40, 0, 7, 0, 0])
    assert lib().amp_device_status(1) == 0


def test_a_decode_step_in_a_graph(cuda, amp_lib):
    s = Server(4, pages=64, width=12)
    s.write([30, 5, 16, 47])
    q, k, v = projection(s.gen, 4)
    cu, one, pos = ints(range(5)), ints([1] * 4), ints(np.zeros((3, 4)))

    def step():
        pos.copy_(s.ctx.expand(3, 4))
        paged.extend_sequences(s.k, s.v, s.table, s.ctx, one, out=s.ctx)
        out = []
        for layer in range(LAYERS):
            qt = paged.rope_append(q, k, v, s.k[layer], s.v[layer], s.table, s.ctx, cu, pos, s.freq, SECTIONS)
            out.append(paged.paged_attn_decode(qt, s.k[layer], s.v[layer], s.table, s.ctx, 12 * 16)[0])
        return out

    state = [x.clone() for x in (s.k, s.v, s.table, s.ctx)]
    eager = [step() for _ in range(20)]
    for x, y in zip((s.k, s.v, s.table, s.ctx), state):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(20):
        graph.replay()
        for a, b in zip(captured, eager[i]):
            assert torch.equal(a, b), i
    torch.cuda.synchronize()
    assert s.ctx.tolist() == [50, 25, 36, 67] and lib().amp_device_status(1) == 0


def test_training_step(cuda, amp_lib):
    lens = [150, 0, 1, 300, 64]
    T = sum(lens)
    gen = torch.Generator().manual_seed(2)
    q, k, v = projection(gen, T)
    do = torch.randn(T, HQ, D, generator=gen).to(torch.bfloat16).cuda()
    cu, f = ints(np.concatenate([[0], np.cumsum(lens)])), freq()
    pos = ints(np.random.default_rng(3).integers(0, 5000, (3, T)))

    def step():
        qt, kt = rope.rope_fwd(q, k, pos, f, SECTIONS)
        o, lse = attention.flash_attn_varlen_fwd(qt, kt, v, cu)
        dqt, dkt, dv = attention.flash_attn_varlen_bwd(qt, kt, v, o, do, lse, cu)
        # the rotation back, in place
        kept = dqt.clone(), dkt.clone()
        dq, dk = rope.rope_bwd(dqt, dkt, pos, f, SECTIONS, out_q=dqt, out_k=dkt)
        return qt, kt, o, lse, *kept, dq, dk, dv

    qt, kt, o, lse, dqt, dkt, dq, dk, dv = first = step()
    check_turn(qt, turned(q, pos, f, SECTIONS, False), HALF[torch.bfloat16])
    want = reference(qt.cpu(), kt.cpu(), v.cpu(), do.cpu(), lens, lens, True)
    check({"o": o, "lse": lse, "dq": dqt, "dk": dkt, "dv": dv}, want, ("o", "lse", "dq", "dk", "dv"))
    check_turn(dq, turned(dqt, pos, f, SECTIONS, False, True), HALF[torch.bfloat16])
    check_turn(dk, turned(dkt, pos, f, SECTIONS, False, True), HALF[torch.bfloat16])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()
    graph.replay()
    for a, b in zip(first, again):
        assert torch.equal(a, b)
