"""Extension of a paged cache whose pages run out, against books kept by hand."""
import random

import books_short_of_pages as short
import pytest
import torch
from test_books_short_of_pages_cpu import walk
from test_gpu_page_books import K, filled, int32, moved, state  # noqa: F401  (a fixture)
from test_gpu_pages import D, generator, normal, pool_of

pytestmark = pytest.mark.gpu


def extended(K, table, lens, refs, add, ps, pools, in_place, more=0):
    """Books and pools after page_extend; `more` further sequences of length 0, that want nothing, make the call one of many"""
    width = len(table[0])
    args = int32(table + [[0] * width] * more), int32(lens + [0] * more), int32(refs)
    kp, vp, ks, vs = pools
    got = K.page_extend(*args, kp, vp, int32(add + [0] * more), page_size=ps, k_scale=ks, v_scale=vs, out=args if in_place else None)
    b = len(table)
    assert not got[0][b:].any() and not got[1][b:].any()
    return got[0][:b], got[1][:b], got[2]


FORMS = [(False, 0), (True, 0), (False, 1100), (True, 1100)]          # in and out of place, by one launch and by two


@pytest.mark.parametrize("in_place,more", FORMS)
def test_two_that_share_the_only_page(K, in_place, more):
    """The first wants a copy and gets none: the second does not write to the page that it lists, and an append leaves the first's tokens as they are."""
    g, ps = generator(1), 16
    (kp, ks), (vp, vs) = pool_of(g, "int8", 2, 1, ps), pool_of(g, "int8", 2, 1, ps)
    start, old = int32([6, 5]), kp.clone()
    table, lens, refs = extended(K, [[0], [0]], [6, 5], [2], [1, 1], ps, (kp, vp, ks, vs), in_place, more)
    assert lens.tolist() == [6, 5] and refs.tolist() == [2] and not table.any()
    new = normal(g, 2, 2, D) * 9
    K.page_append(table, new, new, kp, vp, torch.where(lens > start, start, -1), page_size=ps, k_scale=ks, v_scale=vs)
    assert torch.equal(kp, old)


@pytest.mark.parametrize("in_place,more", FORMS)
@pytest.mark.parametrize("n", [20, 30])
def test_walk(K, n, in_place, more):
    g, ps = generator(n), 4
    k, v = normal(g, 2, n * ps, D), normal(g, 2, n * ps, D)
    for i, ((table, lens, refs), add, (rows, new_lens, new_refs, moves)) in enumerate(walk(n, n, 60)):
        pools = k.clone(), v.clone(), None, None
        got = extended(K, table, lens, refs, add, ps, pools, in_place, more)
        assert got[1].tolist() == new_lens and got[2].tolist() == new_refs and torch.equal(got[0], filled(rows, 10)), i
        assert torch.equal(pools[0], moved(k, None, moves, ps)[0]) and torch.equal(pools[1], moved(v, None, moves, ps)[0])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,most,ps,width,n_pages,left", [(16, 100, 5, 40, 300, 5), (40, 300, 16, 25, 400, 12), (900, 50, 4, 20, 9000, 100), (1100, 50, 4, 20, 9000, 100), (60, 200, 16, 20, 20000, 9)])
def test_many(K, b, most, ps, width, n_pages, left, in_place):
    """`left` pages are free; sequences all want one token."""
    differ = 0
    for seed in range(4):
        table, lens, refs = state(seed, b, most, ps, width, n_pages)
        r = random.Random(seed)
        free = [i for i, x in enumerate(refs) if x == 0]
        for page in r.sample(free, max(0, len(free) - left)):
            refs[page] = 1
        add = [r.choice([1, 1, 1, 0]) for _ in range(b)]
        rows, new_lens, new_refs, _ = short.extend(table, lens, refs, add, ps, width)
        differ += any(a and x == y and x % ps for a, x, y in zip(add, lens, new_lens))
        pools = [normal(generator(seed), 1, n_pages * ps, D) for _ in range(2)] + [None, None]
        got = extended(K, table, lens, refs, add, ps, pools, in_place)
        assert got[1].tolist() == new_lens and got[2].tolist() == new_refs and torch.equal(got[0], filled(rows, width))
    assert differ


@pytest.mark.parametrize("kind", ["f16", "int8"])
def test_prompts_that_there_is_no_room_for(K, kind):
    """As documented: their tokens, several each, go nowhere, and not to the page 0 that their rows of zeros would name."""
    g, ps, n, hkv, lens = generator(5), 16, 4, 2, [30, 40, 10, 20]         # two pages; none for the second, nor for those behind it
    (kp, ks), (vp, vs) = pool_of(g, kind, hkv, n, ps), pool_of(g, kind, hkv, n, ps)
    offsets = int32([0, 30, 70, 80, 100])
    k, v = normal(g, 100, hkv, D), normal(g, 100, hkv, D)
    table, start, refs = torch.zeros((4, 6), dtype=torch.int32, device="cuda"), int32([0] * 4), int32([0] * n)
    table, now, refs = K.page_extend(table, start, refs, kp, vp, int32(lens), page_size=ps, k_scale=ks, v_scale=vs)
    assert now.tolist() == [30, 0, 0, 0] and refs.tolist() == [1, 1, 0, 0]
    one_k, one_v, scales = kp.clone(), vp.clone(), dict(k_scale=None if ks is None else ks.clone(), v_scale=None if vs is None else vs.clone())
    K.page_append(table[:1], k[:30], v[:30], one_k, one_v, start[:1], page_size=ps, offsets=offsets[:2], **scales)
    K.page_append(table, k, v, kp, vp, torch.where(now > start, start, -(1 << 30)), page_size=ps, offsets=offsets, k_scale=ks, v_scale=vs)
    assert torch.equal(kp, one_k) and torch.equal(vp, one_v) and (ks is None or torch.equal(ks, scales["k_scale"]) and torch.equal(vs, scales["v_scale"]))
