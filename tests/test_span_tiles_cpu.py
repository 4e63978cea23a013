"""Which tiles of keys the blocks of prompt attention go through, with documents and prefixes and without, compiled for the host, against the mask key by key."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spec_mcts_b200", "csrc")
SOURCE = r"""
#include <cstdint>
#include "attn_tiles.cuh"
using namespace q40::window::tc;
struct Call { int S, offset, window, sinks, splits, n_documents, prefix; const int32_t *documents, *prefixes; };
static Span span_at(const Call& a, int row) { return a.documents ? span_in(a, row, [&](int k) { return a.documents[k]; }) : span_of(a, row); }
extern "C" int block(const Call* a, int row0, int split, int backwards, int* tiles, int* some, int* all) {
  const int n = smaller(2 * BQ, a->S - row0);
  Span at[4];
  for (int e = 0; e < 4; ++e) at[e] = span_at(*a, row0 + edge_row(e, n));
  const SpanPlaces p(*a, row0, split, at, backwards != 0);
  for (int j = 0; j < p.tiles.n; ++j) {
    tiles[j] = p.tiles.tile(j);
    for (int i = 0; i < 2; ++i) some[2 * j + i] = p.sees[i].some(tiles[j]), all[2 * j + i] = p.sees[i].all(tiles[j]);
  }
  return p.tiles.n;
}
extern "C" int plain_block(const Call* a, int row0, int split, int, int* tiles, int* some, int* all) {
  const Tiles t(*a, row0, 2 * BQ, split);
  const Sees sees[2] = {t.sees(0, BQ, *a), t.sees(BQ, BQ, *a)};
  for (int j = 0; j < t.n; ++j) {
    tiles[j] = t.tile(j);
    for (int i = 0; i < 2; ++i) some[2 * j + i] = sees[i].some(tiles[j]), all[2 * j + i] = sees[i].all(tiles[j]);
  }
  return t.n;
}
extern "C" void span(const Call* a, int row, int* start, int* last) {
  const Span at = span_at(*a, row);
  *start = at.start, *last = at.last;
}
"""


class Call(ctypes.Structure):
    _fields_ = [(x, ctypes.c_int) for x in ("S", "offset", "window", "sinks", "splits", "n_documents", "prefix")] + [(x, ctypes.POINTER(ctypes.c_int32)) for x in ("documents", "prefixes")]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    where = tmp_path_factory.mktemp("span_tiles")
    source, lib = where / "span_tiles.cpp", where / "span_tiles.so"
    source.write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-o", str(lib), str(source)], check=True)
    return ctypes.CDLL(str(lib))


@pytest.fixture
def block(host):
    return host.block


@pytest.fixture
def span(host):
    return host.span


def mask(s, offset, window, sinks, documents, prefixes, prefix):
    n = offset + s
    start, end, pre = np.arange(n), np.arange(n), np.zeros(n, dtype=np.int64)
    for i, (a, b) in enumerate(zip(documents, documents[1:]) if documents is not None else [(0, n)]):
        a, b = max(a, 0), min(b, n)
        start[a:b], end[a:b], pre[a:b] = a, b, prefixes[i] if prefixes is not None else prefix
    start, end, pre = (x[offset:, None] for x in (start, end, pre))
    i, j = np.arange(offset, n)[:, None], np.arange(n)[None]
    return (j >= start) & (j < end) & ((j <= i) | (j - start < pre)) & ((i - j < window) | (j - start < sinks))


def look(block, s, offset=0, window=1 << 29, sinks=0, documents=None, prefixes=None, prefix=0, splits=(1,)):
    whole, int32 = offset + s, lambda x: None if x is None else (ctypes.c_int32 * max(1, len(x)))(*x)
    window, sinks, prefix = min(window, whole), min(sinks, whole), min(prefix, whole)
    seen = mask(s, offset, window, sinks, documents, prefixes, prefix)
    docs, pres = int32(documents), int32(prefixes)
    numbers = lambda n: (ctypes.c_int * n)()
    for row0 in range(0, s, 256):
        for k in splits:
            call = Call(s, offset, window, sinks, k, len(documents) - 1 if documents is not None else 0, prefix, docs, pres)
            for backwards in (0, 1):
                listed = []
                for split in range(k):
                    tiles, some, every = numbers(whole // 128 + 2), numbers(2 * (whole // 128 + 2)), numbers(2 * (whole // 128 + 2))
                    n = block(ctypes.byref(call), row0, split, backwards, tiles, some, every)
                    listed += list(tiles[:n])
                    for j in range(n):
                        assert some[2 * j] or some[2 * j + 1], "a tile that nobody goes through"
                        for i in range(2):
                            part = seen[row0 + 128 * i:min(row0 + 128 * (i + 1), s), 128 * tiles[j]:128 * (tiles[j] + 1)]
                            assert some[2 * j + i] or not part.any()
                            assert not (some[2 * j + i] and every[2 * j + i]) or (part.shape[1] == 128 and part.all())
                assert len(set(listed)) == len(listed)
                rows = seen[row0:row0 + 256]
                assert {t for t in range((whole + 127) // 128) if rows[:, 128 * t:128 * (t + 1)].any()} <= set(listed)


@pytest.mark.parametrize("s,documents,prefix,splits", [(1024, [400, 1024], 0, (1, 2, 4)), (2048, [400, 2048], 1500, (1, 4)), (700, [256, 700], 0, (1, 2)), (512, [130, 131, 500], 0, (1, 2)), (1300, [1200, 1210], 60, (1,)),
                                                       (4000, [0, 1000], 0, (1,)), (600, [599, 600], 0, (1,)), (600, [128, 600], 0, (1, 3)), (385, [384, 385], 0, (1,)), (385, [500], 0, (1,))])
@pytest.mark.parametrize("window,sinks", [(1 << 29, 0), (100, 0), (30, 300), (1, 1)])
def test_rows_in_front_and_behind(block, s, documents, prefix, splits, window, sinks):
    look(block, s, 0, window, sinks, documents, None, prefix, splits)


@pytest.mark.parametrize("seed", range(40))
def test_of_every_kind(block, seed):
    r = random.Random(seed)
    log = lambda most: int(round(2 ** r.uniform(0, np.log2(most))))
    for _ in range(25):
        s = log(1500)
        window, sinks, splits = r.choice([1 << 29, log(s), log(300)]), r.choice([0, log(300), log(8)]), (1, r.randint(2, 6))
        if r.random() < 0.25:
            look(block, s, r.choice([0, log(1000)]), window, sinks, None, None, r.choice([0, log(s), 1 << 29]), splits)
            continue
        n = r.choice([0, 1, 2, 5, log(60)])
        documents = sorted(r.choice([r.randint(0, s), r.randint(-20, s + 20), 128 * r.randint(0, s // 128)]) for _ in range(n + 1))
        if r.random() < 0.5:
            documents[0], documents[-1] = min(documents[0], 0), max(documents[-1], s)
        prefixes = [r.choice([0, -3, log(s), s]) for _ in range(n)] if r.random() < 0.5 else None
        look(block, s, 0, window, sinks, documents, prefixes, r.choice([0, log(s)]) if prefixes is None else 0, splits)


EXTREMES = [-(1 << 31), -(1 << 31) + 1, -1000, -1, 0, 1, 5, 100, 300, 511, 512, 700, 1 << 20, 1 << 30, (1 << 31) - 1]


def test_entries_out_of_range_stay_in_range(span):
    """Spans, tiles and rows that are looked into, whatever the entries are: all within the call's rows."""
    r = random.Random(5)
    for _ in range(4000):
        s, n = r.choice([1, 130, 512]), r.choice([0, 1, 2, 3, 6])
        documents, prefixes = [r.choice(EXTREMES) for _ in range(n + 1)], [r.choice(EXTREMES) for _ in range(n)]
        int32 = lambda x: (ctypes.c_int32 * max(1, len(x)))(*x)
        prefix = r.choice([0, s])
        call = Call(s, 0, r.choice([1, s]), r.choice([0, s]), 1, n, prefix, int32(documents), int32(prefixes) if r.random() < 0.6 else None)
        for row in range(0, s, r.randint(1, 40)):
            start, last = ctypes.c_int(), ctypes.c_int()
            span(ctypes.byref(call), row, ctypes.byref(start), ctypes.byref(last))
            assert 0 <= start.value <= row and (last.value in (-2, row - 1) or row <= last.value < s), (documents, row, start.value, last.value)


def test_documents_that_do_not_rise(block):
    """A tile of keys that a block goes through is gone through by one of its tiles of queries at least, whatever the entries are: who copies it is waited for."""
    r, numbers = random.Random(6), lambda n: (ctypes.c_int * n)()
    for _ in range(3000):
        s, n = r.choice([1, 100, 129, 300, 1100]), r.choice([0, 1, 2, 3, 9])
        documents = [r.choice([r.choice(EXTREMES), r.randint(-50, s + 50)]) for _ in range(n + 1)]
        prefixes = [r.choice([r.choice(EXTREMES), r.randint(0, s)]) for _ in range(n)]
        int32 = lambda x: (ctypes.c_int32 * max(1, len(x)))(*x)
        call = Call(s, 0, r.choice([1, 50, s]), r.choice([0, 5, s]), 1, n, r.choice([0, s]), int32(documents), int32(prefixes) if r.random() < 0.6 else None)
        for row0 in range(0, s, 256):
            tiles, some, every = numbers(s // 128 + 2), numbers(2 * (s // 128 + 2)), numbers(2 * (s // 128 + 2))
            got = block(ctypes.byref(call), row0, 0, r.choice([0, 1]), tiles, some, every)
            assert 0 <= got <= s // 128 + 1 and all(0 <= tiles[j] <= (s - 1) // 128 and (some[2 * j] or some[2 * j + 1]) for j in range(got)), (documents, prefixes, row0)


@pytest.mark.parametrize("seed", range(20))
def test_windows(host, seed):
    """The form without documents and prefixes."""
    r = random.Random(seed)
    log = lambda most: int(round(2 ** r.uniform(0, np.log2(most))))
    for _ in range(25):
        s = log(1500)
        look(host.plain_block, s, r.choice([0, log(1500)]), r.choice([1 << 29, log(s), log(300)]), r.choice([0, log(300), log(8)]), splits=(1, r.randint(2, 6)))
