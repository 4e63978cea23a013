"""What the entry points of changed scores and of a paged cache's books refuse, before anything is enqueued; the books kept by hand against themselves."""
import ctypes
import random

import books_by_hand as hand
import pytest

from spec_mcts_b200._lib import lib

NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5
_buf = ctypes.create_string_buffer(4096)
A = (ctypes.addressof(_buf) + 255) // 256 * 256
NAN = float("nan")


def prompt(q=A, ldq=512, k=A, ldk=256, v=A, ldv=256, o=A, ldo=512, S=4, H=4, Hkv=2, D=128, off=0, w=3, s=0, cap=0.0, slopes=None, docs=None, nd=0, pre=None, prefix=0, keep=0, ws=None, n=0, err=A):
    return lib.q40_attn_causal_scores(q, ldq, k, ldk, v, ldv, o, ldo, S, H, Hkv, D, off, w, s, cap, slopes, docs, nd, pre, prefix, keep, ws, n, err, None)


@pytest.mark.parametrize("status,bad", [(NULL, dict(o=None)), (NULL, dict(err=None)), (NULL, dict(pre=A)), (UNSUPPORTED, dict(D=64)), (SHAPE, dict(H=5)), (SHAPE, dict(w=0)), (SHAPE, dict(s=-1)),
                                        (SHAPE, dict(off=-1)), (SHAPE, dict(off=1 << 30)), (SHAPE, dict(ldq=511)), (SHAPE, dict(cap=-1.0)), (SHAPE, dict(cap=0.009)), (SHAPE, dict(cap=1001.0)),
                                        (SHAPE, dict(cap=NAN)), (SHAPE, dict(prefix=-1)), (SHAPE, dict(docs=A, nd=-1)), (SHAPE, dict(docs=A, nd=1, off=1)), (ALIGN, dict(ldk=260)), (ALIGN, dict(v=A + 8)),
                                        (ALIGN, dict(o=A + 2)), (ALIGN, dict(slopes=A + 2)), (ALIGN, dict(docs=A + 1, nd=1)), (ALIGN, dict(docs=A, nd=1, pre=A + 2)), (ALIGN, dict(err=A + 2)), (0, dict(S=0)),
                                        (WORKSPACE, dict(S=100, off=4000, w=4100, ws=A, n=64)), (ALIGN, dict(S=100, off=4000, w=4100, ws=A + 4, n=1 << 30))])
def test_prompt_refuses(status, bad):
    assert prompt(**bad) == status


def test_prompt_workspace():
    need = lambda S, H, off, w, s=0: lib.q40_attn_causal_scores_workspace_bytes(S, H, H, 128, off, w, s)
    row = 130 * 4
    assert need(1, 32, 0, 1) == need(0, 32, 5000, 5000) == need(100, 32, 5000, 0) == need(5000, 32, 0, 5000) == 0
    assert need(100, 32, 5000, 4096) == 4 * 100 * 32 * row and need(100, 1, 1 << 20, 1 << 20) == 16 * 100 * row


def token(tbl=A, idx=4, tstride=8, lens=A, q=A, qs=512, k=A, v=A, ks=A, vs=A, kind=1, o=A, P=128, B=2, L=128, H=4, Hkv=2, D=128, ps=16, w=0, s=0, cap=5.0, slopes=A, ws=None, n=0):
    return lib.q40_attn_pages_scores(tbl, idx, tstride, lens, q, qs, k, v, ks, vs, kind, o, P, B, L, H, Hkv, D, ps, w, s, cap, slopes, ws, n, None)


@pytest.mark.parametrize("status,bad", [(NULL, dict(q=None)), (NULL, dict(ks=None)), (SHAPE, dict(H=5)), (SHAPE, dict(cap=-5.0)), (SHAPE, dict(cap=2000.0)), (SHAPE, dict(cap=NAN)), (ALIGN, dict(slopes=A + 2)),
                                        (ALIGN, dict(q=A + 8)), (UNSUPPORTED, dict(D=64)), (UNSUPPORTED, dict(kind=3)), (0, dict(B=0)), (WORKSPACE, dict(L=1 << 20, tstride=1 << 16))])
def test_token_refuses(status, bad):
    assert token(**bad) == status


B2, C2 = A + 1024, A + 2048


def fork(t=A, ld=8, lens=A, refs=A, parents=A, to=B2, ldo=8, lo=B2, ro=B2, B=2, W=8, n=16, ps=16, ws=None, nb=0):
    return lib.q40_page_fork(t, ld, lens, refs, parents, to, ldo, lo, ro, B, W, n, ps, ws, nb, None)


def extend(t=A, ld=8, lens=A, refs=A, add=A, to=B2, ldo=8, lo=B2, ro=B2, B=2, W=8, n=16, ps=16, k=A, v=A, ks=A, vs=A, kind=1, P=256, heads=2, ws=C2, nb=1 << 20):
    return lib.q40_page_extend(t, ld, lens, refs, add, to, ldo, lo, ro, B, W, n, ps, k, v, ks, vs, kind, P, heads, ws, nb, None)


def compact(t=A, ld=8, lens=A, refs=A, to=B2, ldo=8, ro=B2, where=B2, B=2, W=8, n=16, ps=16, k=A, v=A, ks=A, vs=A, kind=1, P=256, heads=2, ws=C2, nb=1 << 20):
    return lib.q40_page_compact(t, ld, lens, refs, to, ldo, ro, where, B, W, n, ps, k, v, ks, vs, kind, P, heads, ws, nb, None)


BOOKS = [(NULL, dict(t=None)), (NULL, dict(to=None)), (NULL, dict(lens=None)), (NULL, dict(refs=None)), (NULL, dict(ro=None)), (SHAPE, dict(ld=7)), (SHAPE, dict(ldo=7)), (SHAPE, dict(B=-1)), (SHAPE, dict(W=-1)),
         (SHAPE, dict(W=1 << 29, ld=1 << 29, ldo=1 << 29)), (SHAPE, dict(n=-1)), (SHAPE, dict(n=(1 << 28) + 1)), (SHAPE, dict(ps=0)), (SHAPE, dict(ps=(1 << 29) + 1)), (ALIGN, dict(t=A + 2)), (ALIGN, dict(lens=A + 1)),
         (ALIGN, dict(refs=A + 2)), (ALIGN, dict(to=B2 + 2)), (ALIGN, dict(ro=B2 + 1))]
POOLS = [(NULL, dict(k=None)), (NULL, dict(vs=None)), (SHAPE, dict(P=255)), (SHAPE, dict(P=240)), (SHAPE, dict(heads=-1)), (UNSUPPORTED, dict(kind=3)), (UNSUPPORTED, dict(kind=-1)), (ALIGN, dict(v=A + 8)),
         (ALIGN, dict(ks=A + 2)), (WORKSPACE, dict(to=A, ws=None)), (ALIGN, dict(ws=C2 + 4)), (WORKSPACE, dict(to=A, nb=15)), (WORKSPACE, dict(n=16385, ps=1, P=16385, nb=15)), (SHAPE, dict(to=A, ldo=9))]


@pytest.mark.parametrize("status,bad", BOOKS + [(NULL, dict(parents=None)), (NULL, dict(lo=None)), (ALIGN, dict(parents=A + 2)), (ALIGN, dict(lo=A + 2)), (ALIGN, dict(ws=A + 2)), (SHAPE, dict(to=A, ldo=9)), (WORKSPACE, dict(to=A, B=600)), (WORKSPACE, dict(lo=A, B=600, ws=C2, nb=600 * 36 - 1)),
                                                (0, dict(B=0, n=0))])
def test_fork_refuses(status, bad):
    assert fork(**bad) == status


@pytest.mark.parametrize("status,bad", BOOKS + POOLS + [(NULL, dict(add=None)), (NULL, dict(lo=None)), (ALIGN, dict(add=A + 2)), (SHAPE, dict(B=16385)), (0, dict(B=0, n=0))])
def test_extend_refuses(status, bad):
    assert extend(**bad) == status


@pytest.mark.parametrize("status,bad", BOOKS + POOLS + [(NULL, dict(where=None)), (ALIGN, dict(where=B2 + 2))])
def test_compact_refuses(status, bad):
    assert compact(**bad) == status


def test_books_workspace():
    assert lib.q40_page_fork_workspace_bytes(600, 8, 16) == 600 * 9 * 4 and lib.q40_page_fork_workspace_bytes(500, 8, 16) == 0
    assert lib.q40_page_extend_workspace_bytes(10, 100, 1) == (70 + 200 + 4) * 4 and lib.q40_page_extend_workspace_bytes(-1, 5, 1) == 0
    assert lib.q40_page_extend_workspace_bytes(10, 100, 0) == lib.q40_page_extend_workspace_bytes(1024, 16384, 0) == 0 < lib.q40_page_extend_workspace_bytes(1025, 1, 0)
    assert lib.q40_page_compact_workspace_bytes(101, 1) == (3 * 51 + 4) * 4 and lib.q40_page_compact_workspace_bytes(-1, 1) == 0
    assert lib.q40_page_compact_workspace_bytes(16384, 0) == 0 < lib.q40_page_compact_workspace_bytes(16385, 0)


def test_hand_kept_books_stay_consistent():
    """References count what is listed, no page that is written to is shared, and pages in use are the first ones after a compaction."""
    r, ps, width, n = random.Random(1), 4, 10, 70
    rows, lens, refs = [[] for _ in range(9)], [0] * 9, [0] * n
    flat = lambda: [x + [0] * (width - len(x)) for x in rows]
    count = lambda: [sum(x.count(i) for x in rows) for i in range(n)]
    for _ in range(200):
        rows, lens, refs = hand.fork(flat(), lens, refs, [r.choice([i, i, i, r.randrange(9), -1]) for i in range(9)], ps)
        assert refs == count()
        was, old = lens, [list(x) for x in rows]
        rows, lens, refs, moves = hand.extend(flat(), lens, refs, [r.choice([1, 1, 2, -1, 0, 9]) for _ in range(9)], ps, width)
        assert refs == count() and all(hand.pages(x, ps) == len(y) for x, y in zip(lens, rows))
        for b in range(9):
            if lens[b] > was[b]:
                assert all(refs[page] == 1 for page in rows[b][was[b] // ps:])
                assert [dict((y, x) for x, y, _ in moves).get(page, page) for page in rows[b][:len(old[b])]] == old[b]
        rows, refs, where, moves = hand.compact(flat(), lens, refs, ps)
        assert refs == count() and all(refs[:sum(x > 0 for x in refs)])
