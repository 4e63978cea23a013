"""The books of a paged cache, kept by hand, while pages run out."""
import random

import books_by_hand as hand
import books_short_of_pages as short
import pytest


def walk(seed, n, steps=200, ps=4, width=10, b=9):
    """Forks, extensions and compactions in turn; before and after each extension: rows, lengths, references"""
    r = random.Random(seed)
    rows, lens, refs = [[] for _ in range(b)], [0] * b, [0] * n
    flat = lambda: [x + [0] * (width - len(x)) for x in rows]
    for _ in range(steps):
        rows, lens, refs = hand.fork(flat(), lens, refs, [r.choice([i, i, i, r.randrange(b), -1]) for i in range(b)], ps)
        add = [r.choice([1, 1, 2, -1, 0, 9]) for _ in range(b)]
        before = flat(), lens, refs
        rows, lens, refs, moves = short.extend(*before, add, ps, width)
        yield before, add, (rows, lens, refs, moves)
        rows, refs, _, _ = hand.compact(flat(), lens, refs, ps)


@pytest.mark.parametrize("n", [70, 30, 20, 8])
def test_no_page_that_is_written_to_is_listed_by_another(n):
    refused, ps, width = 0, 4, 10
    for seed in range(20):
        for (table, was, old), add, (rows, lens, refs, moves) in walk(seed, n):
            assert refs == [sum(x.count(i) for x in rows) for i in range(n)] and all(hand.pages(x, ps) == len(y) for x, y in zip(lens, rows))
            copy_of = {dst: src for src, dst, _ in moves}
            for b in range(9):
                if lens[b] > was[b]:
                    assert all(refs[page] == 1 for page in rows[b][was[b] // ps:])
                    assert [copy_of.get(page, page) for page in rows[b][:hand.pages(was[b], ps)]] == table[b][:hand.pages(was[b], ps)]
                elif add[b] > 0:
                    assert lens[b] == was[b] and rows[b] == table[b][:hand.pages(was[b], ps)]
                    refused += hand.pages(was[b] + add[b], ps) <= width
    assert (refused == 0) == (n == 70)


def test_as_before_where_none_is_refused():
    for (table, lens, refs), add, got in walk(1, 70):
        assert hand.extend(table, lens, refs, add, 4, 10) == got


def test_two_that_share_the_only_page():
    """The first is longer: what the second wrote behind its five tokens would be the first's sixth."""
    table, lens, refs = [[0], [0]], [6, 5], [2]
    assert short.extend(table, lens, refs, [1, 1], 16, 1) == ([[0], [0]], lens, refs, [])
    assert short.extend(table, lens, refs + [0], [1, 1], 16, 1) == ([[1], [0]], [7, 6], [1, 1], [(0, 1, 6)])
