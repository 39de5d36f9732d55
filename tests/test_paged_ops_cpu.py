"""Refusals of the paged cache's bookkeeping: argument errors return before any CUDA work."""
import pytest

from amp_b200._lib import AmpError, call

P, W = 1 << 20, 1 << 40   # an aligned address that is never read; a workspace large enough


def copy(k=P, v=P, layers=1, pages=9, H=2, D=64, src=P, dst=P, n=3, ws=P, wb=W):
    call("amp_paged_copy_pages_dev", k, v, layers, pages, H, D, src, dst, n, ws, wb, None)


def fork(k=P, v=P, layers=1, pages=9, H=2, D=64, table=P, ctx=P, rows=4, width=3, parents=P, children=P,
         n=2, done=P, ws=P, wb=W):
    call("amp_paged_fork_dev", k, v, layers, pages, H, D, table, ctx, rows, width, parents, children, n,
         done, ws, wb, None)


def extend(k=P, v=P, layers=1, pages=9, H=2, D=64, table=P, ctx=P, rows=4, width=3, add=P, out=P, done=P,
           ws=P, wb=W):
    call("amp_paged_extend_dev", k, v, layers, pages, H, D, table, ctx, rows, width, add, out, done, ws, wb,
         None)


def compact(k=P, v=P, layers=1, pages=9, H=2, D=64, table=P, ctx=P, rows=4, width=3, out=P, used=P, ws=P,
            wb=W):
    call("amp_paged_compact_dev", k, v, layers, pages, H, D, table, ctx, rows, width, out, used, ws, wb, None)


def free(table=P, ctx=P, rows=4, width=3, seqs=P, n=2):
    call("amp_paged_free_dev", table, ctx, rows, width, seqs, n, None)


POOLS = [(dict(k=None), -1), (dict(v=None), -1), (dict(k=P + 8), -1), (dict(layers=0), -1),
         (dict(pages=0), -1), (dict(H=0), -1), (dict(D=0), -1), (dict(pages=1 << 20), -2),
         (dict(H=1 << 20, D=1 << 10), -2)]
TABLE = [(dict(table=None), -1), (dict(ctx=None), -1), (dict(rows=0), -1), (dict(width=0), -1),
         (dict(rows=1 << 20), -2), (dict(width=1 << 25), -2)]
SPACE = [(dict(ws=None), -1), (dict(ws=P + 4), -1), (dict(wb=8), -1)]


@pytest.mark.parametrize("entry,kw,code", [
    *((copy, *x) for x in POOLS), (copy, dict(src=None), -1), (copy, dict(dst=None), -1),
    (copy, dict(n=-1), -1), *((fork, *x) for x in POOLS), (fork, dict(parents=None), -1),
    (fork, dict(children=None), -1), (fork, dict(done=None), -1), (fork, dict(n=-1), -1),
    *((extend, *x) for x in POOLS), *((compact, *x) for x in POOLS),
    *((free, *x) for x in TABLE[2:4]), (free, dict(n=-1), -1), (free, dict(table=None), -1),
    (free, dict(rows=1 << 20), -2)], ids=lambda x: getattr(x, "__name__", str(x)))
def test_refused_arguments(entry, kw, code, amp_lib):
    with pytest.raises(AmpError) as e:
        entry(**kw)
    assert e.value.code == code


@pytest.mark.parametrize("entry", [fork, extend, compact])
@pytest.mark.parametrize("kw,code", TABLE[:4], ids=str)
def test_refused_tables(entry, kw, code, amp_lib):
    with pytest.raises(AmpError) as e:
        entry(**kw)
    assert e.value.code == code


@pytest.mark.parametrize("entry", [copy, fork, extend, compact])
@pytest.mark.parametrize("kw,code", SPACE, ids=str)
def test_refused_workspaces(entry, kw, code, amp_lib):
    with pytest.raises(AmpError) as e:
        entry(**kw)
    assert e.value.code == code


def test_nothing_to_do(amp_lib):
    copy(n=0, src=None, ws=None)
    fork(n=0, parents=None, ws=None)
    free(n=0, seqs=None)


def test_workspace_sizes(amp_lib):
    assert amp_lib.amp_paged_copy_workspace_bytes(10) >= 80
    assert amp_lib.amp_paged_fork_workspace_bytes(10, 100) >= 4 * 10 * 102
    assert amp_lib.amp_paged_extend_workspace_bytes(10, 100) >= 400
    assert amp_lib.amp_paged_compact_workspace_bytes(100) >= 800
    assert amp_lib.amp_paged_copy_workspace_bytes(-1) == 0
    assert amp_lib.amp_paged_fork_workspace_bytes(1, 0) == 0


@pytest.mark.parametrize("kw", [dict(add=P + 16, out=P + 16, done=P), dict(add=P + 16, done=P + 16, out=P),
                                dict(out=P + 16, done=P + 16), dict(ctx=P + 16, done=P + 16, out=P + 32)], ids=str)
def test_extend_refuses_results_in_each_others_place(kw, amp_lib):
    with pytest.raises(AmpError, match="share memory") as e:
        extend(**kw)
    assert e.value.code == -1
