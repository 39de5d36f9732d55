"""The paged cache's bookkeeping on the B200 against a plain model: equal tables, lengths, pages."""
import numpy as np
import pytest
import torch

from paged_model import Cache
from amp_b200 import paged
from amp_b200._lib import lib

pytestmark = pytest.mark.gpu


class Both:
    """A cache on the device and its model, run side by side."""

    def __init__(self, ctx, spare=8, layers=2, Hkv=2, D=64, seed=0, width=None):
        rng = np.random.default_rng(seed)
        ctx = np.asarray(ctx, np.int32)
        need = -(-ctx // 16)
        pages = max(1, int(need.sum()) + spare)
        order, at = rng.permutation(pages), 0
        table = np.full((len(ctx), width or max(1, int(need.max())) + 3), -1, np.int32)
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        shape = (layers, pages, Hkv, 16, D)
        self.k, self.v = (torch.randint(-30000, 30000, shape, dtype=torch.int16, device="cuda").view(torch.bfloat16)
                          for _ in range(2))
        self.table, self.ctx = torch.from_numpy(table).cuda(), torch.from_numpy(ctx).cuda()
        self.model = Cache(table, ctx, *(x.view(torch.int16).cpu().numpy() for x in (self.k, self.v)))

    def pools(self):
        return self.k, self.v

    def check(self):
        m = self.model
        assert (lib().amp_device_status(1) == -1) == m.bad
        m.bad = False
        ctx = self.ctx.cpu().numpy()
        assert np.array_equal(ctx, m.ctx)
        table = self.table.cpu().numpy()
        for r, c in enumerate(ctx):
            assert np.array_equal(table[r, :m.need(c)], m.table[r, :m.need(c)]), r
        for x, y in ((self.k, m.k), (self.v, m.v)):
            assert np.array_equal(x.view(torch.int16).cpu().numpy(), y)

    def copy(self, src, dst):
        paged.copy_pages(*self.pools(), ints(src), ints(dst))
        self.model.copy(src, dst)
        self.check()

    def fork(self, parents, children):
        done = paged.fork_sequences(*self.pools(), self.table, self.ctx, ints(parents), ints(children))
        assert np.array_equal(done.cpu().numpy(), self.model.fork(parents, children))
        self.check()
        for c in set(children):   # a child's row says -1 past its pages
            if 0 <= c < len(self.model.ctx) and list(children).count(c) == 1:
                assert (self.table[c, self.model.need(self.model.ctx[c]):] == -1).all() or c in parents
        return done.cpu().numpy()

    def extend(self, add, in_place=True):
        out, done = paged.extend_sequences(*self.pools(), self.table, self.ctx, ints(add),
                                           out=self.ctx if in_place else None)
        self.ctx = out
        want = self.model.extend(add)
        assert np.array_equal(done.cpu().numpy(), want)
        self.check()
        return want

    def compact(self, in_place=False):
        out, used = paged.compact_pages(*self.pools(), self.table, self.ctx, out=self.table if in_place else None)
        self.table = out
        assert used.item() == self.model.compact()
        self.check()
        assert np.array_equal(out.cpu().numpy(), self.model.table)

    def free(self, seqs):
        paged.free_sequences(self.table, self.ctx, ints(seqs))
        self.model.free(seqs)
        self.check()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def test_copy(cuda, amp_lib):
    c = Both([200], spare=20)
    c.copy([0, 1, 2], [20, 21, 22])
    c.copy([5], [5])
    c.copy([-1, 3, 4, 7], [3, -1, 30, 7])
    c.copy([], [])


def test_copy_of_pages_named_twice_is_skipped_and_reported(cuda, amp_lib):
    c = Both([200], spare=20)
    c.copy([0, 1, 2], [20, 20, 21])            # one target twice
    c.copy([0, 5, 6], [5, 22, 23])             # a source that is another's target
    c.copy([0, 5, 6], [33, 24, 10 ** 6])       # outside the pool
    c.copy([8, 8, 9], [8, 25, 9])              # onto itself: still a source


def test_pages_past_32_bits(cuda, amp_lib):
    Hkv, D = 8, 128
    pages = (1 << 32) // (Hkv * 16 * D) + 64          # the last pages start past 2^32 elements
    k, v = (torch.zeros(pages, Hkv, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    last = pages - 1
    k[last], v[last] = 1.0, 2.0
    paged.copy_pages(k, v, ints([last, 0]), ints([last - 7, last - 9]))
    assert (k[last - 7] == 1.0).all() and (v[last - 7] == 2.0).all() and not k[last - 9].any()
    table, ctx = ints([[last, last - 7, -1], [3, -1, -1]]), ints([20, 5])
    assert paged.fork_sequences(k, v, table, ctx, ints([0]), ints([1])).all()
    assert table.tolist() == [[last, last - 7, -1], [last, 0, -1]] and (k[0] == 1.0).all()
    new, used = paged.compact_pages(k, v, table, ctx)
    assert new.tolist() == [[2, 1, -1], [2, 0, -1]] and used.item() == 3 and (v[:3] == 2.0).all()


@pytest.mark.parametrize("n", [300, 1024, 1025, 3000])
def test_copy_of_many_pages(n, cuda, amp_lib):
    """Few pairs are compared by the copying blocks, many by a plan: the same pages are left alone."""
    rng = np.random.default_rng(n)
    c = Both([16], spare=4000, layers=1, Hkv=1, D=8)
    order = rng.permutation(c.model.pages)
    src, dst = rng.choice(order[:900], n), order[900:900 + n].copy()
    c.copy(src, dst)                            # a source may be named often
    dst[::7] = dst[rng.permutation(n)[:len(dst[::7])]]   # some targets twice
    src[::50] = dst[1::50][:len(src[::50])]              # some sources are targets
    src[3::90], dst[5::80] = -1, 10 ** 7
    c.copy(src, dst)


def test_copy_many_layers_and_large_pages(cuda, amp_lib):
    c = Both([3000], spare=300, layers=3, Hkv=8, D=128)
    rng = np.random.default_rng(1)
    order = rng.permutation(c.model.pages)
    c.copy(order[:200], order[200:400])


def test_fork_shares_full_pages_and_copies_the_last(cuda, amp_lib):
    c = Both([40, 32, 1, 0, 0, 0, 0, 0])
    c.fork([0, 1, 2, 3, 0], [4, 5, 6, 7, 3])   # row 3 (empty) is a parent and a child
    assert c.table[4, 0] == c.table[0, 0] and c.table[4, 2] != c.table[0, 2]
    c.fork([0], [0])
    c.fork([], [])


def test_fork_replaces_what_the_child_held(cuda, amp_lib):
    c = Both([40, 100, 50, 7], spare=0)        # a full pool: only the children's pages are free
    c.fork([0, 0], [1, 2])
    c.fork([3, 3, 3], [0, 1, 2])


def test_fork_chains_and_swaps(cuda, amp_lib):
    c = Both([40, 100, 50, 7, 20])
    c.fork([0, 1, 2, 3, 4], [1, 2, 3, 4, 0])   # every row is both
    c.fork([1, 0], [0, 1])


def test_fork_without_pages_left(cuda, amp_lib):
    c = Both([17, 32, 5, 0, 0, 0, 0], spare=1)
    done = c.fork([0, 1, 2, 0], [3, 4, 5, 6])
    assert list(done) == [1, 1, 0, 0]


def test_fork_of_bad_rows_and_children_named_twice(cuda, amp_lib):
    c = Both([40, 32, 1, 9, 0, 0])
    done = c.fork([0, 9, -1, 1, 2, 3], [4, 5, 5, 3, 3, -7])
    assert list(done) == [1, 0, 0, 0, 0, 0]


def test_extend(cuda, amp_lib):
    c = Both([0, 1, 16, 17, 31, 32], spare=40, width=12)
    c.extend([1, 15, 1, 0, 1, 60])
    c.extend([16, 1, 200, -1, 0, 3], in_place=False)   # too long for the table; negative
    c.extend([0] * 6)


def test_extend_without_pages_left(cuda, amp_lib):
    c = Both([16, 16, 3, 16], spare=3, width=40)
    assert list(c.extend([17, 40, 2, 1])) == [1, 0, 1, 0]


def test_extend_copies_a_shared_last_page(cuda, amp_lib):
    c = Both([64, 0, 0], spare=10)
    c.fork([0, 0], [1, 2])                     # shares four full pages
    short = ints([40, 40, 64])                 # two rows step back into a shared page
    c.ctx.copy_(short)
    c.model.ctx[:] = [40, 40, 64]
    c.extend([1, 30, 1])
    assert len({c.table[r, 2].item() for r in range(3)}) == 3


def test_extend_long_prompts(cuda, amp_lib):
    c = Both([5] * 40, spare=6000, Hkv=1, layers=1, width=300)
    c.extend([100 * i for i in range(40)])


@pytest.mark.parametrize("in_place", [False, True])
def test_compact(in_place, cuda, amp_lib):
    c = Both([400, 30, 1, 0, 160, 90], spare=50, seed=3)
    c.fork([0], [3])
    c.free([4, 1])
    c.compact(in_place)
    c.compact(in_place)                        # nothing to move any more
    c.extend([5] * 6)


def test_compact_of_an_empty_and_of_a_full_pool(cuda, amp_lib):
    c = Both([0, 0], spare=5)
    c.compact()
    c = Both([320], spare=0)
    c.compact()


def test_free_twice_and_out_of_range(cuda, amp_lib):
    c = Both([40, 30, 20])
    c.free([1, 1])
    c.free([7, -1, 0])
    c.free([])


def test_table_entries_outside_the_pool_are_reported(cuda, amp_lib):
    for bad in (-1, 10 ** 6):
        c = Both([40, 30, 0, 0], spare=9)
        c.table[0, 2] = bad
        c.model.table[0, 2] = bad
        c.fork([0, 1], [2, 3])
        c = Both([40, 30, 50], spare=9)
        c.table[0, 1] = bad
        c.model.table[0, 1] = bad
        c.compact()


@pytest.mark.parametrize("seed", range(6))
def test_random_runs(seed, cuda, amp_lib):
    rng = np.random.default_rng(seed)
    rows = int(rng.integers(1, 40))
    c = Both(rng.integers(0, 200, rows), spare=int(rng.integers(0, 200)), seed=seed,
             layers=int(rng.integers(1, 3)), Hkv=int(rng.integers(1, 4)), D=int(rng.choice([8, 64])), width=20)
    for _ in range(12):
        op = rng.choice(["fork", "extend", "compact", "free"])
        if op == "fork":
            n = int(rng.integers(0, rows + 1))
            c.fork(rng.integers(0, rows, n), rng.permutation(rows)[:n])
        elif op == "extend":
            c.extend(rng.integers(0, 60, rows) * (rng.random(rows) < 0.6))
        elif op == "compact":
            c.compact()
        else:
            c.free(rng.integers(0, rows, 2))


def test_more_rows_and_pages_than_one_pass(cuda, amp_lib):
    rng = np.random.default_rng(9)
    n = 2500
    c = Both(np.concatenate([rng.integers(1, 300, n), np.zeros(n, int)]), spare=60000, layers=1, Hkv=1, D=8, width=20)
    c.fork(rng.integers(0, n, n), n + rng.permutation(n))
    c.extend(rng.integers(0, 20, 2 * n))
    c.free(rng.permutation(2 * n)[:n])
    c.compact()


def test_graph_and_other_stream(cuda, amp_lib):
    a, b = (Both([40, 100, 7, 0, 0, 0], spare=30, seed=5) for _ in range(2))
    b.k.copy_(a.k), b.v.copy_(a.v)
    parents, children, add = ints([0, 1, 2]), ints([3, 4, 5]), ints([1, 20, 3, 1, 1, 9])

    def step(c):
        paged.fork_sequences(*c.pools(), c.table, c.ctx, parents, children)
        paged.extend_sequences(*c.pools(), c.table, c.ctx, add, out=c.ctx)
        return paged.compact_pages(*c.pools(), c.table, c.ctx, out=c.table)

    step(a)
    state = [x.clone() for x in (b.k, b.v, b.table, b.ctx)]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        step(b)
    torch.cuda.synchronize()
    assert torch.equal(a.table, b.table) and torch.equal(a.ctx, b.ctx)
    assert torch.equal(a.k.view(torch.int16), b.k.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for x, y in zip((b.k, b.v, b.table, b.ctx), state):
        x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.table, b.table) and torch.equal(a.v.view(torch.int16), b.v.view(torch.int16))


def test_python_refuses(cuda, amp_lib):
    c = Both([40, 0])
    k, v = c.pools()
    one = ints([0])
    for call in (lambda: paged.copy_pages(k, v[:1], one, one), lambda: paged.copy_pages(k, v, one, ints([0, 1])),
                 lambda: paged.copy_pages(k, v, one.long(), one), lambda: paged.copy_pages(k.float(), v, one, one),
                 lambda: paged.copy_pages(k.transpose(0, 1), v, one, one),
                 lambda: paged.fork_sequences(k, v, c.table, c.ctx[:1], one, one),
                 lambda: paged.fork_sequences(k, v, c.table[:, ::2], c.ctx, one, one),
                 lambda: paged.extend_sequences(k, v, c.table, c.ctx, one),
                 lambda: paged.compact_pages(k, v, c.table, c.ctx, out=c.table[:, :1]),
                 lambda: paged.fork_sequences(k, v, c.table, c.ctx, one, one,
                                              workspace=torch.empty(4, dtype=torch.uint8, device="cuda")),
                 lambda: paged.free_sequences(c.table.cpu(), c.ctx.cpu(), one.cpu())):
        with pytest.raises(ValueError):
            call()


def test_extend_does_not_write_lengths_over_what_it_adds(cuda, amp_lib):
    """Two rows share a partly filled page, so each has to get a copy: with the lengths in add's place
    the plan saw rows without tokens."""
    pool = torch.zeros(8, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[3, -1], [3, -1]], dtype=torch.int32, device="cuda")
    ctx, add = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([5, 5], [1, 2]))
    before = table.clone()
    with pytest.raises(RuntimeError, match="share memory"):
        paged.extend_sequences(pool, pool.clone(), table, ctx, add, out=add)
    assert torch.equal(table, before) and add.tolist() == [1, 2]
    new, done = paged.extend_sequences(pool, pool.clone(), table, ctx, add, out=ctx)
    assert new.tolist() == [6, 7] and done.tolist() == [1, 1] and table[:, 0].tolist() == [0, 1]


@pytest.mark.parametrize("n,layers,Hkv,D", [(300, 4, 1, 64), (300, 3, 1, 64), (300, 4, 2, 128), (1025, 1, 1, 64)])
def test_copy_of_many_pairs_by_either_way(n, layers, Hkv, D, cuda, amp_lib):
    """Around the limits between comparing pairs in place and planning them, with pairs that clash."""
    pages = 4 * n
    g = torch.Generator("cuda").manual_seed(n + layers)
    pools = [torch.randn(layers, pages, Hkv, 16, D, device="cuda", generator=g).bfloat16() for _ in range(2)]
    perm = torch.randperm(pages, device="cuda", generator=g).int()
    src, dst = perm[:n].clone(), perm[n:2 * n].clone()
    src[1], dst[2], src[3] = -1, -5, dst[3]                # nothing to do
    want = [p.clone() for p in pools]
    real = [0] + list(range(4, n))
    for w in want:
        w[:, dst[real].long()] = w[:, src[real].long()]
    paged.copy_pages(*pools, src, dst)
    assert all(map(torch.equal, pools, want)) and lib().amp_device_status(1) == 0
    dst[7], src[9] = dst[6], dst[8]                        # two onto one page; one from a page that is written
    dst[10] = pages
    keep = [0, 4, 5, 8] + list(range(11, n))
    want = [p.clone() for p in pools]
    for w in want:
        w[:, dst[keep].long()] = w[:, src[keep].long()]
    paged.copy_pages(*pools, src, dst)
    assert all(map(torch.equal, pools, want))
    assert lib().amp_device_status(1) == -1 and lib().amp_device_status(1) == 0


@pytest.mark.parametrize("rows,layers", [(2, 32), (3, 5), (40, 7)])
def test_extend_copies_shared_pages_in_every_layer(rows, layers, cuda, amp_lib):
    """More blocks copy than there are rows: each row gets its own copy, whatever the layer."""
    g = torch.Generator("cuda").manual_seed(rows)
    pools = [torch.randn(layers, 2 * rows, 8, 16, 128, device="cuda", generator=g).bfloat16() for _ in range(2)]
    before = [p.clone() for p in pools]
    last = 2 * rows - 1
    table, ctx, add = (torch.full((rows, 2), -1), torch.full((rows,), 9), torch.ones(rows))
    table[:, 0] = last
    table, ctx, add = (x.int().cuda() for x in (table, ctx, add))
    new, done = paged.extend_sequences(*pools, table, ctx, add)
    assert new.tolist() == [10] * rows and done.tolist() == [1] * rows
    assert table[:, 0].tolist() == list(range(rows))
    for p, b in zip(pools, before):
        assert torch.equal(p[:, :rows], b[:, last:].expand(-1, rows, -1, -1, -1))
        assert torch.equal(p[:, rows:], b[:, rows:])
    assert lib().amp_device_status(1) == 0
