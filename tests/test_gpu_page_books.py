"""Forks, extension and compaction of a paged cache against books kept by hand."""
import math
import random

import books_by_hand as hand
import pytest
import torch
from test_gpu_pages import D, WEIGHT, generator, normal, pool_of, tables
from test_gpu_scores import attention, slopes_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from spec_mcts_b200 import kernels
    return kernels


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def state(seed, b, most, ps, width, n_pages, held=0):
    """Sequences of up to `most` tokens that share pages at random, and `held` pages that are in use by none of them."""
    r = random.Random(seed)
    ids = list(range(n_pages))
    r.shuffle(ids)
    rows, lens = [], []
    for i in range(b):
        like = r.randrange(i) if i and r.random() < 0.6 else None
        n = r.randint(0, most)
        if like is not None and r.random() < 0.5:
            n = lens[like]                                # as it came out of a fork
        keep = 0 if like is None else min(hand.pages(n, ps), len(rows[like]), r.randint(0, 100) if n != lens[like] else 1 << 30)
        if keep + max(0, hand.pages(n, ps) - keep) > keep and hand.pages(n, ps) - keep > len(ids) - held:
            n = keep * ps
        row = (rows[like][:keep] if keep else []) + [ids.pop() for _ in range(hand.pages(n, ps) - keep)]
        rows.append(row)
        lens.append(n)
    refs = [0] * n_pages
    for row in rows:
        for page in row:
            refs[page] += 1
    for _ in range(min(held, len(ids))):
        refs[ids.pop()] = r.randint(1, 3)
    table = [row + [r.randrange(-5, n_pages + 5) for _ in range(width - len(row))] for row in rows]      # left over behind them
    return table, lens, refs


def filled(rows, width):
    return int32([row + [0] * (width - len(row)) for row in rows]).view(len(rows), width)


def moved(pool, scale, moves, ps):
    pool, scale = pool.clone(), None if scale is None else scale.clone()
    x = pool.view(torch.uint8) if scale is not None else pool
    old, old_scale = x.clone(), None if scale is None else scale.clone()
    for a, b, n in moves:
        x[..., b * ps:b * ps + n, :] = old[..., a * ps:a * ps + n, :]
        if scale is not None:
            scale[..., b] = old_scale[..., a]
    return x, scale


SIZES = [(1, 40, 16, 5, 20), (3, 7, 1, 9, 40), (16, 100, 5, 40, 300), (40, 300, 16, 25, 400), (130, 60, 64, 3, 500), (1100, 50, 4, 20, 9000), (7, 3000, 2, 1600, 30000), (600, 90, 16, 7, 200_000)]
KINDS = ["f16", "int8", "e4m3"]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,most,ps,width,n_pages", SIZES)
def test_fork(K, b, most, ps, width, n_pages, in_place):
    for seed in range(3):
        table, lens, refs = state(seed, b, most, ps, width, n_pages, 3)
        r = random.Random(seed)
        parents = [r.choice([i, i, -1, b, 1 << 30, r.randrange(b), r.randrange(b)]) for i in range(b)]
        if seed == 2:
            parents = [b - 1 - i for i in range(b)]       # all in turn
        rows, new_lens, new_refs = hand.fork(table, lens, refs, parents, ps)
        args = int32(table), int32(lens), int32(refs)
        got = K.page_fork(*args, int32(parents), page_size=ps, out=args if in_place else None)
        assert torch.equal(got[0], filled(rows, width)) and got[1].tolist() == new_lens and got[2].tolist() == new_refs
        assert in_place == (got[0].data_ptr() == args[0].data_ptr())
        if not in_place:
            assert args[0].tolist() == table and args[1].tolist() == lens and args[2].tolist() == refs


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,most,ps,width,n_pages", SIZES)
def test_extend(K, b, most, ps, width, n_pages, in_place):
    for seed in range(6):
        kind, layers = KINDS[seed % 3], [1, 3][seed % 2]
        table, lens, refs = state(seed, b, most, ps, width, n_pages, [2, n_pages][seed == 4])
        r = random.Random(seed)
        add = [r.choice([0, 1, 1, 1, 1, r.randint(-most, most), r.randint(-3, 3 * ps), 1 << 31 - 1, -(1 << 31)]) for _ in range(b)]
        add = [min(x, (1 << 31) - 1) for x in add]
        if seed == 5:
            add = [1] * b
        rows, new_lens, new_refs, moves = hand.extend(table, lens, refs, add, ps, width)
        g = generator(seed)
        (kp, ks), (vp, vs) = pool_of(g, kind, 2 * layers, n_pages if n_pages < 50000 else 1, ps), pool_of(g, kind, 2 * layers, n_pages if n_pages < 50000 else 1, ps)
        if n_pages >= 50000:                              # many pages of small pools: heads of none
            kp, vp = kp[:0].new_zeros((0, n_pages * ps, D)), vp[:0].new_zeros((0, n_pages * ps, D))
            ks, vs = (None if s is None else s.new_zeros((0, n_pages)) for s in (ks, vs))
        want = [moved(kp, ks, moves, ps), moved(vp, vs, moves, ps)]
        if layers > 1 and kp.shape[0]:
            kp, vp = kp.view(layers, 2, -1, D), vp.view(layers, 2, -1, D)
            ks, vs = (None if s is None else s.view(layers, 2, -1) for s in (ks, vs))
        args = int32(table), int32(lens), int32(refs)
        got = K.page_extend(*args, kp, vp, int32(add), page_size=ps, k_scale=ks, v_scale=vs, out=args if in_place else None)
        assert got[1].tolist() == new_lens and got[2].tolist() == new_refs and torch.equal(got[0], filled(rows, width))
        for pool, scale, (x, s) in ((kp, ks, want[0]), (vp, vs, want[1])):
            assert torch.equal(pool.view(x.dtype).view_as(x), x) and (s is None or torch.equal(scale.view_as(s), s))
        if not in_place:
            assert args[0].tolist() == table and args[1].tolist() == lens and args[2].tolist() == refs


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,most,ps,width,n_pages", SIZES[:-1] + [(1, 0, 16, 1, 31), (1, 0, 16, 1, 33), (2, 4000, 1, 4000, 8192)])
def test_compact(K, b, most, ps, width, n_pages, in_place):
    for seed in range(3):
        kind, layers = KINDS[seed % 3], [1, 3][seed % 2]
        table, lens, refs = state(seed, b, most, ps, width, n_pages, [3, n_pages, n_pages // 3][seed])
        rows, new_refs, where, moves = hand.compact(table, lens, refs, ps)
        g = generator(seed)
        (kp, ks), (vp, vs) = pool_of(g, kind, layers, n_pages, ps), pool_of(g, kind, layers, n_pages, ps)
        want = [moved(kp, ks, moves, ps), moved(vp, vs, moves, ps)]
        args, out = (int32(table), int32(lens), int32(refs)), None
        if in_place:
            out = args[0], args[2], torch.empty_like(args[2])
        got = K.page_compact(*args, kp, vp, page_size=ps, k_scale=ks, v_scale=vs, out=out)
        assert torch.equal(got[0], filled(rows, width)) and got[1].tolist() == new_refs and got[2].tolist() == where
        for pool, scale, (x, s) in ((kp, ks, want[0]), (vp, vs, want[1])):
            # what has moved away lies where it was until it is written over
            assert torch.equal(pool.view(x.dtype), x) and (s is None or torch.equal(scale, s))
        if not in_place:
            assert args[0].tolist() == table and args[2].tolist() == refs


@pytest.mark.parametrize("in_place", [(), (0,), (1,), (2,), (0, 1, 2)])
def test_much_that_moves_and_books_partly_in_place(K, in_place):
    """Pools of many layers, whose pages more than a cluster moves; some of the books in place."""
    b, ps, width, n_pages, heads = 60, 16, 20, 500, 40
    table, lens, refs = state(8, b, 200, ps, width, n_pages, 100)
    add = [1 + i % 2 for i in range(b)]
    g = generator(3)
    (kp, ks), (vp, vs) = pool_of(g, "e4m3", heads, n_pages, ps), pool_of(g, "e4m3", heads, n_pages, ps)
    fresh = lambda: [int32(table), int32(lens), int32(refs)]

    def out_of(args, which):
        return tuple(args[i] if n in in_place else torch.full_like(args[i], 9) for n, i in enumerate(which))

    rows, new_lens, new_refs = hand.fork(table, lens, refs, [i // 3 for i in range(b)], ps)
    args = fresh()
    got = K.page_fork(*args, int32([i // 3 for i in range(b)]), page_size=ps, out=out_of(args, (0, 1, 2)))
    assert torch.equal(got[0], filled(rows, width)) and got[1].tolist() == new_lens and got[2].tolist() == new_refs
    rows, new_lens, new_refs, moves = hand.extend(table, lens, refs, add, ps, width)
    assert len(moves) > 10
    pools, args = (kp.clone(), vp.clone(), ks.clone(), vs.clone()), fresh()
    got = K.page_extend(*args, *pools[:2], int32(add), page_size=ps, k_scale=pools[2], v_scale=pools[3], out=out_of(args, (0, 1, 2)))
    assert torch.equal(got[0], filled(rows, width)) and got[1].tolist() == new_lens and got[2].tolist() == new_refs
    for pool, scale, old, old_scale in zip(pools[:2], pools[2:], (kp, vp), (ks, vs)):
        x, s = moved(old, old_scale, moves, ps)
        assert torch.equal(pool.view(x.dtype), x) and torch.equal(scale, s)
    rows, new_refs, where, moves = hand.compact(table, lens, refs, ps)
    assert len(moves) > 10
    pools, args = (kp.clone(), vp.clone(), ks.clone(), vs.clone()), fresh()
    out = out_of(args, (0, 2)) + (torch.empty_like(args[2]),)
    got = K.page_compact(*args, *pools[:2], page_size=ps, k_scale=pools[2], v_scale=pools[3], out=out)
    assert torch.equal(got[0], filled(rows, width)) and got[1].tolist() == new_refs and got[2].tolist() == where and all(a is b for a, b in zip(got, out))
    for pool, scale, old, old_scale in zip(pools[:2], pools[2:], (kp, vp), (ks, vs)):
        x, s = moved(old, old_scale, moves, ps)
        assert torch.equal(pool.view(x.dtype), x) and torch.equal(scale, s)


def test_sequences_that_want_more_than_there_is(K):
    """More than 2^31 pages in all: the first that does not get its own, and those behind it that want any, stay as they are."""
    b, ps, width = 40, 1, 1 << 20
    table = torch.zeros((b, width), dtype=torch.int32, device="cuda")
    lens, refs, add = [0] * b, [0] * 50, [1] * 5 + [1 << 20] * 30 + [0, 1, -3, 1, 2]
    pool = torch.zeros((1, 50, D), dtype=torch.float16, device="cuda")
    got = K.page_extend(table, int32(lens), int32(refs), pool, pool.clone(), int32(add), page_size=ps)
    assert got[1].tolist() == [1] * 5 + [0] * 35 and got[0][:5, 0].tolist() == list(range(5)) and got[2].tolist() == [1] * 5 + [0] * 45
    add[5:35] = [(1 << 31) - 1] * 30                      # ... and than the table has room for: these want nothing, and others do
    got = K.page_extend(table, int32(lens), int32(refs), pool, pool.clone(), int32(add), page_size=ps)
    assert got[1].tolist() == [1] * 5 + [0] * 31 + [1, 0, 1, 2] and got[2].tolist() == [1] * 9 + [0] * 41


def test_most_sequences(K):
    b = 16384
    table, lens = torch.zeros((b, 1), dtype=torch.int32, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
    pool = torch.zeros((1, b, D), dtype=torch.float16, device="cuda")
    got = K.page_extend(table, lens, torch.zeros(b, dtype=torch.int32, device="cuda"), pool, pool.clone(), torch.ones_like(lens), page_size=1)
    assert torch.equal(got[0][:, 0], torch.arange(b, dtype=torch.int32, device="cuda")) and (got[1] == 1).all() and (got[2] == 1).all()
    with pytest.raises(K.Q40Error):
        more = torch.zeros(b + 1, dtype=torch.int32, device="cuda")
        K.page_extend(more[:, None], more, more, pool, pool, more, page_size=1)


def test_nothing(K):
    pool = torch.zeros((2, 64, D), dtype=torch.float16, device="cuda")
    for b, w, n in ((0, 4, 4), (3, 0, 4), (0, 0, 0), (2, 3, 0)):
        books = torch.ones((b, w), dtype=torch.int32, device="cuda"), torch.full((b,), 5, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
        some = torch.zeros(b, dtype=torch.int32, device="cuda")
        fork, more, less = K.page_fork(*books, some, page_size=16), K.page_extend(*books, pool, pool, some, page_size=16), K.page_compact(*books, pool, pool, page_size=16)
        assert fork[0].shape == more[0].shape == less[0].shape == (b, w) and less[2].tolist() == list(range(n))
        assert more[2].tolist() == [1] * n


def test_books_that_do_not_fit_fault_nothing(K):
    """Ids out of range, lengths that no table has room for, references that are wrong: what comes is undefined, and the next call is right."""
    g, ps, n = generator(1), 16, 64
    (kp, ks), (vp, vs) = pool_of(g, "int8", 2, n, ps), pool_of(g, "int8", 2, n, ps)
    r = random.Random(3)
    for _ in range(8):
        wild = lambda: r.choice([-(1 << 31), -1, 0, 1, 5, 63, 64, 1 << 20, (1 << 31) - 1, r.randrange(64), r.randrange(64)])
        books = [int32([[wild() for _ in range(9)] for _ in range(30)]), int32([wild() for _ in range(30)]), int32([r.choice([-3, 0, 0, 1, 1, 2, 7]) for _ in range(n)])]
        for out in (None, tuple(books)):
            K.page_fork(*books, int32([wild() for _ in range(30)]), page_size=ps, out=out)
            K.page_extend(*books, kp, vp, int32([wild() for _ in range(30)]), page_size=ps, k_scale=ks, v_scale=vs, out=out)
            K.page_compact(*books, kp, vp, page_size=ps, k_scale=ks, v_scale=vs, out=out and (books[0], books[2], torch.empty_like(books[2])))
        torch.cuda.synchronize()
    test_extend(K, 16, 100, 5, 40, 300, False)


def test_numbers_of_other_types(K):
    """Wide ones out of range are so, and not what their low bits say."""
    table, lens, refs = state(2, 9, 40, 4, 12, 90)
    pool = lambda: normal(generator(1), 1, 360, D)
    wide = lambda *x: torch.tensor(x, dtype=torch.int64, device="cuda")
    books = int32(table), int32(lens), int32(refs)
    far = K.page_fork(*books, wide(1 << 32, -(1 << 40), (1 << 33) + 1, 3, 4, 5, 6, 7, 8), page_size=4)
    near = K.page_fork(*books, int32([-1, -1, -1, 3, 4, 5, 6, 7, 8]), page_size=4)
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    far = K.page_extend(*books, pool(), pool(), wide(1 << 32, -(1 << 40), (1 << 33) + 1, 1, 1, 1, 0, 0, 0), page_size=4)
    near = K.page_extend(*books, pool(), pool(), int32([1 << 30, -(1 << 30), 1 << 30, 1, 1, 1, 0, 0, 0]), page_size=4)
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    short = K.page_extend(*books, pool(), pool(), int32([1, -1, 0, 1, 1, 1, 0, 0, 0]).short(), page_size=4)
    assert all(torch.equal(a, b) for a, b in zip(short, K.page_extend(*books, pool(), pool(), int32([1, -1, 0, 1, 1, 1, 0, 0, 0]), page_size=4)))


def test_strided_books(K):
    table, lens, refs = state(5, 20, 60, 4, 16, 200)
    wide = torch.full((20, 50), 9, dtype=torch.int32, device="cuda")
    wide[:, 3:19] = int32(table)
    parents, add = int32([i ^ 1 for i in range(20)]), int32([i % 5 - 1 for i in range(20)])
    pool = lambda: normal(generator(1), 2, 800, D)
    plain = K.page_fork(int32(table), int32(lens), int32(refs), parents, page_size=4)
    into = torch.full((20, 40), 7, dtype=torch.int32, device="cuda")
    out = into[:, 4:20], torch.empty(20, dtype=torch.int32, device="cuda"), torch.empty(200, dtype=torch.int32, device="cuda")
    got = K.page_fork(wide[:, 3:19], int32(lens), int32(refs), parents, page_size=4, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, plain)) and (into[:, :4] == 7).all() and (into[:, 20:] == 7).all()
    spread = wide[:, 3:19].repeat_interleave(2, 1)[:, ::2]                                            # columns apart
    for call, last in ((K.page_extend, (add,)), (K.page_compact, ())):
        plain = call(int32(table), int32(lens), int32(refs), pool(), pool(), *last, page_size=4)
        for p in (wide[:, 3:19], spread):
            assert all(torch.equal(a, b) for a, b in zip(call(p, int32(lens), int32(refs), pool(), pool(), *last, page_size=4), plain))
    view = wide[:, 3:19]
    got = K.page_extend(view, int32(lens), int32(refs), pool(), pool(), add, page_size=4, out=(view, *out[1:]))
    assert torch.equal(view, K.page_extend(int32(table), int32(lens), int32(refs), pool(), pool(), add, page_size=4)[0]) and (wide[:, :3] == 9).all() and (wide[:, 19:] == 9).all()


def test_refusals(K):
    p, lens, refs = torch.zeros((3, 4), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    pool, codes = torch.zeros((2, 128, D), dtype=torch.float16, device="cuda"), torch.zeros((2, 128, D), dtype=torch.int8, device="cuda")
    scale, where = torch.zeros((2, 8), device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    fork = lambda p=p, lens=lens, refs=refs, parents=lens, ps=16, out=None: K.page_fork(p, lens, refs, parents, page_size=ps, out=out)
    extend = lambda p=p, lens=lens, refs=refs, k=pool, v=pool, add=lens, ps=16, ks=None, vs=None, out=None: K.page_extend(p, lens, refs, k, v, add, page_size=ps, k_scale=ks, v_scale=vs, out=out)
    compact = lambda p=p, lens=lens, refs=refs, k=pool, v=pool, ps=16, ks=None, vs=None, out=None: K.page_compact(p, lens, refs, k, v, page_size=ps, k_scale=ks, v_scale=vs, out=out)
    books = [dict(p=p.short()), dict(p=p.long()), dict(p=p[0]), dict(lens=lens[:2]), dict(lens=lens.long()), dict(refs=refs.long()), dict(refs=refs[None]), dict(ps=0), dict(ps=1 << 30), dict(p=p.cpu()),
             dict(refs=refs.cpu()), dict(out=(p, lens)), dict(out=(p[:, :3], lens, refs)), dict(out=(p, lens.long(), refs)), dict(out=(p.t().contiguous().t(), lens, refs)),
             dict(out=(p, refs[:3], refs)), dict(out=(refs[:12].new_zeros(12).view(3, 4), lens, lens.new_zeros(3)))]
    pools = [dict(k=pool[0]), dict(k=pool[:1]), dict(k=pool[:, :100], v=pool[:, :100]), dict(k=codes, v=codes), dict(k=codes, v=codes, ks=scale, vs=scale[:1]), dict(ks=scale, vs=scale), dict(k=pool.float(), v=pool.float()),
             dict(k=pool[:, :64].contiguous(), v=pool[:, :64].contiguous()), dict(k=pool[..., :64].contiguous(), v=pool[..., :64].contiguous()), dict(k=pool.cpu()), dict(v=codes), dict(k=pool[None])]
    for call, bad in ((fork, books + [dict(parents=lens[:2]), dict(parents=lens.float()), dict(parents=lens.cpu())]), (extend, books + pools + [dict(add=lens[:1]), dict(add=lens.float())]),
                      (compact, [x for x in books if "out" not in x] + pools + [dict(out=(p, refs)), dict(out=(p, refs, refs)), dict(out=(p, where, refs)), dict(out=(p, refs, where[:4]))])):
        for x in bad:
            with pytest.raises(K.Q40Error):
                call(**x)
        call()
    flat = torch.zeros(40, dtype=torch.int32, device="cuda")
    with pytest.raises(K.Q40Error):                       # partly over what is read
        K.page_fork(flat[:12].view(3, 4), lens, refs, lens, page_size=16, out=(flat[4:16].view(3, 4), lens, refs))
    with pytest.raises(K.Q40Error):                       # over the parents, or what is added
        K.page_fork(p, lens, refs, lens, page_size=16, out=(p, lens, refs))
    with pytest.raises(K.Q40Error):
        K.page_extend(p, lens, refs, pool, pool, refs[2:5], page_size=16, out=(p, lens, refs))
    with pytest.raises(K.Q40Error):                       # over other books
        K.page_fork(p, lens, flat[:8], lens, page_size=16, out=(flat[4:16].view(3, 4), lens, where))


def test_captured_and_replayed(K):
    """A step that forks, extends and compacts in place, replayed on what the books are then; another graph beside it."""
    ps, width, n = 4, 12, 120
    stages, g = [state(s, 12, 40, ps, width, n) for s in range(4)], generator(1)
    books, pool, pool2 = [torch.empty_like(int32(x)) for x in stages[0]], normal(g, 2, n * ps, D), normal(g, 2, n * ps, D)
    parents, add, where = int32([i // 2 for i in range(12)]), int32([1 + i % 3 for i in range(12)]), torch.empty(n, dtype=torch.int32, device="cuda")

    def step():
        K.page_fork(*books, parents, page_size=ps, out=tuple(books))
        K.page_extend(*books, pool, pool2, add, page_size=ps, out=tuple(books))
        K.page_compact(*books, pool, pool2, page_size=ps, out=(books[0], books[2], where))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t, x in zip(books, stages[0]):
            t.copy_(int32(x))
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for table, lens, refs in stages:
        for t, x in zip(books, (table, lens, refs)):
            t.copy_(int32(x))
        graph.replay()
        rows, lens, refs = hand.fork(table, lens, refs, parents.tolist(), ps)
        rows, lens, refs, _ = hand.extend([r + [0] * (width - len(r)) for r in rows], lens, refs, add.tolist(), ps, width)
        rows, refs, want, _ = hand.compact([r + [0] * (width - len(r)) for r in rows], lens, refs, ps)
        assert torch.equal(books[0], filled(rows, width)) and books[1].tolist() == lens and books[2].tolist() == refs and where.tolist() == want


@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
def test_a_search_over_a_paged_cache(K, kind):
    """Two prompts in one call, their keys and values to pages, branches of them that share these, tokens of their own, branches given up, pages moved to the front: what branches
    read is what they wrote, and moving pages changes no bit of what is read."""
    h, hkv, ps, width, n_pages, b = 4, 2, 16, 8, 60, 6
    g, softcap, slopes, lens = generator(11), 20.0, slopes_of(4), [37, 50]
    total = sum(lens)
    qkv = normal(g, total, h + 2 * hkv, D)
    q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    cos, sin = (torch.ones((128, 64), dtype=torch.float16, device="cuda"), torch.zeros((128, 64), dtype=torch.float16, device="cuda"))
    documents = int32([0, lens[0], total])
    (kp, ks), (vp, vs) = pool_of(g, kind, hkv, n_pages, ps), pool_of(g, kind, hkv, n_pages, ps)
    scales = dict(k_scale=ks, v_scale=vs)
    books = [torch.zeros((b, width), dtype=torch.int32, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda")]
    history = [[] for _ in range(b)]                      # of each sequence: what its keys and values are

    # the prompts
    o = K.causal_attn(q, k, v, documents=documents, softcap=softcap, slopes=slopes)
    for a, e in ((0, lens[0]), (lens[0], total)):
        one = K.causal_attn(q[a:e], k[a:e], v[a:e], softcap=softcap, slopes=slopes)
        assert (o[a:e].float() - one.float()).abs().max() <= 2 ** -9 * 4
    start = books[1].clone()
    books = list(K.page_extend(*books, kp, vp, int32(lens + [0] * (b - 2)), page_size=ps, **scales))
    K.page_append(books[0][:2], k, v, kp, vp, start[:2], page_size=ps, offsets=documents, **scales)
    for i, (a, e) in enumerate(((0, lens[0]), (lens[0], total))):
        history[i] = [(k[t], v[t]) for t in range(a, e)]

    def read():
        n = books[1].tolist()
        longest = width * ps
        if kind == "f16":
            return K.page_flash_attn(books[0], query, kp, vp, n_pages * ps, b, longest, h, D, page_size=ps, seq_lens=books[1], softcap=softcap, slopes=slopes)
        return K.page_flash_attn_q8(books[0], query, kp, vp, ks, vs, page_size=ps, seq_lens=books[1], softcap=softcap, slopes=slopes)

    for step, parents in enumerate([[0, 1, 0, 1, 0, 1], [0, 1, 2, 3, 4, 5], [2, 2, 2, 5, 5, 5], [0, 0, -1, 3, -1, 5], [1, 0, 3, 3, 3, 3]]):
        books = list(K.page_fork(*books, int32(parents), page_size=ps))
        history = [list(history[p]) if p >= 0 else [] for p in parents]
        start = books[1].clone()
        alive = [p >= 0 and len(history[i]) > 0 for i, p in enumerate(parents)]
        books = list(K.page_extend(*books, kp, vp, int32([int(x) for x in alive]), page_size=ps, **scales))
        assert (books[1] - start).tolist() == [int(x) for x in alive]
        new_k, new_v, query = normal(g, b, hkv, D), normal(g, b, hkv, D), normal(g, b, h, D)
        K.page_append(books[0], new_k, new_v, kp, vp, torch.where(int32([int(x) for x in alive]) > 0, start, -1), page_size=ps, **scales)
        for i in range(b):
            if alive[i]:
                history[i].append((new_k[i], new_v[i]))
        got = read()
        for i in range(b):
            if not history[i]:
                assert not got[i].any()
                continue
            kk, vv = (torch.stack([x[c] for x in history[i]]).double().transpose(0, 1)[:, None] for c in (0, 1))
            n = len(history[i])
            seen, far = torch.ones((1, n), dtype=torch.bool, device="cuda"), (n - 1 - torch.arange(n, device="cuda"))[None]
            want, size, off = attention(query[i:i + 1], kk, vv, seen, far, softcap, slopes)
            # 8 bits: an element is off by half a step of its page's scale, and by as much for each time that the scale grew; a key's by that many of |q| in its score
            coarse = 0 if kind == "f16" else (0.5 / 127 if kind == "int8" else 2 ** -4) * 3
            most = max(kk.abs().max(), vv.abs().max()).item()
            key = coarse * most * query[i].float().norm(dim=-1).double()[None, :, None]      # sum over 128 dims / sqrt(128), by Cauchy-Schwarz
            bound = 2 ** -11 * want.abs() + (WEIGHT + torch.expm1(2 * key)) * size + off + coarse * most + 2 ** -25
            assert ((got[i:i + 1].double() - want).abs() <= bound).all()
        before = read()
        table, refs, where = K.page_compact(*books, kp, vp, page_size=ps, **scales)
        books = [table, books[1], refs]
        used = int((where >= 0).sum())
        assert (refs[:used] > 0).all() and not refs[used:].any() and int(refs.sum()) == sum(hand.pages(x, ps) for x in books[1].tolist())
        assert torch.equal(read(), before)


def test_streams_and_threads_beside_each_other(K):
    """Each with books and prompts of its own."""
    import threading

    def work(seed, results):
        torch.cuda.set_device(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            table, lens, refs = state(seed, 30, 60, 4, 24, 400)
            g = torch.Generator(device="cuda").manual_seed(seed)
            pool, pool2, q = normal(g, 2, 1600, D), normal(g, 2, 1600, D), normal(g, 600, 4, D)
            torch.cuda.current_stream().synchronize()
            for i in range(20):
                books = K.page_fork(int32(table), int32(lens), int32(refs), int32([(b * 7 + i) % 30 for b in range(30)]), page_size=4)
                books = K.page_extend(*books, pool, pool2, int32([b % 3 for b in range(30)]), page_size=4)
                o = K.causal_attn(q, q[:, :2], q[:, 2:], documents=int32([0, 100 + i, 600]), softcap=20.0)
                last = [x.clone() for x in (*books, *K.page_compact(*books, pool, pool2, page_size=4), pool, pool2, o)]
            torch.cuda.current_stream().synchronize()
            results.append(last)

    alone, together = [[] for _ in range(4)], [[] for _ in range(4)]
    for i, r in enumerate(alone):
        work(i, r)
    threads = [threading.Thread(target=work, args=(i, r)) for i, r in enumerate(together)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, y) for a, b in zip(alone, together) for x, y in zip(a[0], b[0]))
