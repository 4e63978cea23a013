"""Attention with capped scores, scores that fall with distance, documents and prefixes, for prompts and for one token over pages, each against its
definition in 64 bits."""
import math

import pytest
import torch
from test_gpu_pages import D, WEIGHT, generator, normal, pool_of, table_of, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from spec_mcts_b200 import kernels
    return kernels


def slopes_of(h):
    return torch.pow(2.0, -8.0 * torch.arange(1, h + 1, dtype=torch.float64) / h).float().cuda()


def attention(q, k, v, seen, far, softcap, slopes):
    """q [rows, H, D], k / v [Hkv, rows or 1, keys, D] in 64 bits, seen and far [rows, keys] -> the result, and what its weights' errors may make of it"""
    b, h, _ = q.shape
    hkv = k.shape[0]
    x = (q.double().view(b, hkv, h // hkv, D).transpose(0, 1) @ k.transpose(-1, -2)) / math.sqrt(D)
    if softcap:
        x = torch.tanh(x / softcap) * softcap
    cost = torch.zeros(1, dtype=torch.float64, device="cuda")
    if slopes is not None:
        cost = slopes.double().view(hkv, 1, h // hkv, 1) * far.double()[None, :, None]
    w = torch.softmax((x - cost).masked_fill(~seen[None, :, None], -math.inf), -1).nan_to_num(0.0)
    v = v.masked_fill(~seen.any(0)[None, None, :, None], 0.0) if v.shape[1] == 1 else v.masked_fill(~seen[None, ..., None], 0.0)
    out, size = w @ v, w @ v.abs()
    # A cap: its polynomial 1.1e-7 and seven roundings, or 2^x and a quotient to 2^-22, of a value up to the cap: 2^-21 of it, in weights and in their sum.  A bias: four
    # roundings of 2^-24 of it, of the products in powers of two and of their sum with a score (2^-22), likewise
    off = 2 * (softcap or 0) * 2 ** -21 * size + 2 ** -22 * ((w * cost.abs()) @ v.abs() + (w * cost.abs()).sum(-1, keepdim=True) * size)
    back = lambda t: t.transpose(0, 1).reshape(b, h, D)
    return back(out), back(size), back(off)


# ---- prompts -------------------------------------------------------------------------------------------------------
def spans(n, documents, prefixes, prefix):
    """Beginning and end of each row's document (both the row: none), and its prefix"""
    start, end, pre = torch.arange(n), torch.arange(n), torch.zeros(n, dtype=torch.long)
    for i, (a, b) in enumerate(zip(documents, documents[1:])):
        a, b = max(a, 0), min(b, n)
        start[a:b], end[a:b], pre[a:b] = a, b, prefixes[i] if prefixes is not None else prefix
    return start.cuda(), end.cuda(), pre.cuda()


def mask(s, offset, window, sinks, documents=None, prefixes=None, prefix=0):
    n = offset + s
    start, end, pre = (x[offset:, None] for x in spans(n, [0, n] if documents is None else documents, prefixes, prefix))
    i, j = torch.arange(offset, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    return (j >= start) & (j < end) & ((j <= i) | (j - start < pre)) & ((i - j < (window or n)) | (j - start < sinks)), (i - j).abs()


def check(got, want, size, off, keys, v):
    # as for a prompt with a window: weights rounded to fp16, 2^-11 of each, or half a step of the smallest, 2^-25 of the largest weight
    bound = 2 ** -11 * want.abs() + (WEIGHT + 2 ** -11) * size + off + keys * 2 ** -25 * v.float().nan_to_num(0, 0, 0).abs().max() + 2 ** -25
    assert ((got.double() - want).abs() <= bound).all()


def run(K, g, s, h, hkv, window=None, sinks=0, offset=0, softcap=None, alibi=False, documents=None, prefixes=None, prefix=0, out=None, size=1.0):
    n = offset + s
    q, k, v = normal(g, s, h, D) * size, normal(g, n + 3, hkv, D), normal(g, n + 3, hkv, D)
    k[n:], v[n:] = math.nan, math.nan                     # rows behind the last position
    int32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    slopes = slopes_of(h) if alibi else None
    got = K.causal_attn(q, k, v, out, window=window, sinks=sinks, offset=offset, softcap=softcap, slopes=slopes, documents=int32(documents),
                        prefix=prefix if prefixes is None else int32(prefixes))
    assert K.tc_error_flag() == 0
    seen, far = mask(s, offset, window, sinks, documents, prefixes, prefix)
    wide = lambda x: x[:n].double().transpose(0, 1)[:, None]
    check(got, *attention(q, wide(k), wide(v), seen, far, softcap, slopes), n, v)
    return got, seen


SIZES = [(1, 2, 1, None, 0, 0), (2, 4, 4, 1, 0, 0), (77, 8, 2, None, 0, 0), (127, 2, 2, 50, 3, 5), (128, 2, 1, None, 0, 128), (129, 3, 3, 129, 0, 0), (256, 2, 2, None, 0, 1),
         (257, 5, 1, 100, 140, 300), (700, 4, 2, 333, 4, 0), (1025, 2, 1, None, 0, 0), (1, 4, 2, 900, 5, 3000), (100, 2, 2, None, 0, 2500)]


@pytest.mark.parametrize("softcap,alibi", [(50.0, False), (2.0, False), (None, True), (30.0, True)])
@pytest.mark.parametrize("s,h,hkv,window,sinks,offset", SIZES)
def test_scores(K, s, h, hkv, window, sinks, offset, softcap, alibi):
    run(K, generator(s + h), s, h, hkv, window, sinks, offset, softcap, alibi)


@pytest.mark.parametrize("softcap", [0.01, 0.5, 5.0, 1000.0])
@pytest.mark.parametrize("size", [0.01, 1.0, 30.0, 200.0])
def test_caps_of_every_size(K, softcap, size):
    """Scores far below and far above the cap, and both in one tile."""
    g = generator(3)
    run(K, g, 300, 4, 2, softcap=softcap, size=size)


@pytest.mark.parametrize("prefix,window,sinks,offset", [(1, None, 0, 0), (2, None, 0, 0), (100, None, 0, 0), (128, 40, 0, 0), (129, None, 0, 0), (200, 1, 3, 0), (299, 64, 130, 0), (300, None, 0, 0),
                                                        (5000, None, 0, 0), (250, None, 0, 100), (90, 30, 2, 100), (400, 200, 0, 100)])
@pytest.mark.parametrize("softcap,alibi", [(None, False), (20.0, True)])
def test_prefix(K, prefix, window, sinks, offset, softcap, alibi):
    run(K, generator(prefix), 300, 4, 2, window, sinks, offset, softcap, alibi, prefix=prefix)


DOCUMENTS = [[0, 300], [0, 1, 2, 3, 300], [0, 0, 0, 150, 150, 300, 300], [0, 128, 256, 300], [0, 127, 255, 257, 300], [40, 41, 170, 290], [299, 300], [100, 100], [0, 0], [300, 300], [150],
             [0, 5, 11, 18, 90, 91, 140, 200, 260, 299], list(range(0, 301, 4)), [260, 300], [0, 20], [0, 129], [0, 299, 400]]


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (30, 2), (10, 200), (1000, 5)])
@pytest.mark.parametrize("documents", DOCUMENTS)
def test_documents(K, documents, window, sinks):
    got, seen = run(K, generator(len(documents)), 300, 4, 2, window, sinks, documents=documents)
    assert not got[~seen.any(1)].any()


@pytest.mark.parametrize("softcap,alibi,window", [(None, False, None), (50.0, False, 70), (None, True, None), (5.0, True, 200)])
@pytest.mark.parametrize("documents,prefixes", [([0, 40, 300], [10, 100]), ([0, 128, 384, 400, 1000], [128, 200, 0, 600]), ([5, 700, 990], [0, 1000]), ([0, 1, 2, 999], [1, -5, 1 << 30]), ([0, 400, 999], [-(1 << 31), (1 << 31) - 1]),
                                                ([0, 500, 1000], [499, 2])])
def test_documents_with_prefixes(K, documents, prefixes, softcap, alibi, window):
    run(K, generator(7), 1000, 2, 1, window, 3 if window else 0, 0, softcap, alibi, documents, prefixes)
    run(K, generator(8), 1000, 2, 1, window, 0, 0, softcap, alibi, documents, None, 60)


def test_many_documents(K):
    """More than the rows of a tile, empty ones among them."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 4, (1500,), generator=g)
    run(K, generator(2), int(lens.sum()), 2, 2, documents=[0] + lens.cumsum(0).tolist())


def test_one_document_is_none(K):
    """And positions in front of it are none of its."""
    g = generator(5)
    q, k, v = normal(g, 700, 4, D), normal(g, 700, 2, D), normal(g, 700, 2, D)
    plain = K.causal_attn(q, k, v, window=700)
    one = K.causal_attn(q, k, v, documents=torch.tensor([0, 700], dtype=torch.int32, device="cuda"))
    assert torch.equal(plain, one)
    apart = K.causal_attn(q, k, v, documents=torch.tensor([256, 700], dtype=torch.int32, device="cuda"))
    # (not the bits of a call of the 444: how CTAs share keys goes by the number of rows)
    seen, far = mask(444, 0, None, 0)
    wide = lambda x: x[256:].double().transpose(0, 1)[:, None]
    check(apart[256:], *attention(q[256:], wide(k), wide(v), seen, far, None, None), 444, v)
    assert not apart[:256].any()


@pytest.mark.parametrize("s", [90, 700, 2500])
def test_rows_of_no_document_stay_as_they_are(K, s):
    """In `out`, also where CTAs share keys."""
    g = generator(6)
    qkv, out = normal(g, s, 4, D), torch.full((s, 3, D), 7.0, dtype=torch.float16, device="cuda")
    q, k, v = qkv[:, :2], qkv[:, 2:3], qkv[:, 3:]
    a, b = 30, s - 40
    documents = torch.tensor([a, a, b], dtype=torch.int32, device="cuda")
    got = K.causal_attn(q, k, v, out[:, 1:], documents=documents)
    assert got.data_ptr() == out[:, 1:].data_ptr() and (out[:, 0] == 7).all() and (got[:a] == 7).all() and (got[b:] == 7).all()
    fresh = K.causal_attn(q, k, v, documents=documents)
    assert torch.equal(fresh[a:b], got[a:b]) and not fresh[:a].any() and not fresh[b:].any()


def test_offsets_that_do_not_rise_fault_nothing(K):
    """Their results are undefined; the call ends, and the next is right."""
    g = generator(9)
    q, k, v = normal(g, 600, 2, D), normal(g, 600, 1, D), normal(g, 600, 1, D)
    for bad in ([500, 3, 400, 20, 600], [-(1 << 31), (1 << 31) - 1], [0, 1 << 30, 7], [600, 500, 0], [-5, -1]):
        K.causal_attn(q, k, v, documents=torch.tensor(bad, dtype=torch.int32, device="cuda"), prefix=1 << 30, window=200, sinks=600)
        assert K.tc_error_flag() == 0
    run(K, g, 300, 2, 1, documents=[0, 100, 300])


@pytest.mark.parametrize("softcap,alibi", [(None, False), (10.0, True)])
def test_values_that_are_not_finite(K, softcap, alibi):
    """They reach the queries that see them, and no other; so do keys."""
    g = generator(12)
    s, documents, prefixes = 700, [0, 200, 650], [150, 20]
    q, k, v = normal(g, s, 4, D), normal(g, s, 2, D), normal(g, s, 2, D)
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    slopes = slopes_of(4) if alibi else None
    call = lambda: K.causal_attn(q, k, v, softcap=softcap, slopes=slopes, documents=int32(documents), prefix=int32(prefixes))
    seen, _ = mask(s, 0, None, 0, documents, prefixes)
    for j in (0, 149, 199, 200, 649, 660):
        kept = v.clone()
        v[j, 0, 5], v[j, 1, 9] = math.inf, math.nan
        got = call()
        assert ((got[:, :2, 5] == math.inf) == seen[:, j, None]).all() and (got[:, 2:, 9].isnan() == seen[:, j, None]).all()
        got[:, :2, 5], got[:, 2:, 9] = 0, 0
        assert got.isfinite().all()
        v.copy_(kept)
    k[300] = math.nan
    got = call()
    assert (got[..., 0].isnan() == seen[:, 300, None]).all()


def test_infinite_scores_are_capped(K):
    g = generator(13)
    q, k, v = normal(g, 64, 2, D), normal(g, 64, 2, D), normal(g, 64, 2, D)
    q[:, :, 0], k[:, :, 0] = 1.0, 0.0
    k[3, :, 0], k[4, :, 0] = math.inf, -math.inf
    got = K.causal_attn(q, k, v, softcap=5.0)
    x = torch.tanh(torch.einsum("ihd,jhd->hij", q.double(), k.double()) / math.sqrt(D) / 5) * 5
    x = x.masked_fill(~torch.ones(64, 64, dtype=torch.bool, device="cuda").tril(), -math.inf)
    want = torch.einsum("hij,jhd->ihd", torch.softmax(x, -1), v.double())
    assert ((got.double() - want).abs() <= 2 ** -11 * want.abs() + (WEIGHT + 2 ** -10) * 4.5 + 1e-6).all()


def test_steep_slopes(K):
    """Down to a key's weight of nothing, and up, where the farthest key has it all; a slope of its own for each head."""
    g = generator(14)
    s = 900
    q, k, v = normal(g, s, 4, D), normal(g, s, 4, D), normal(g, s, 4, D)
    slopes = torch.tensor([100.0, -3.0, 0.0, 1e-4], device="cuda")
    got = K.causal_attn(q, k, v, slopes=slopes)
    seen, far = mask(s, 0, None, 0)
    wide = lambda x: x.double().transpose(0, 1)[:, None]
    check(got, *attention(q, wide(k), wide(v), seen, far, None, slopes), s, v)
    assert torch.equal(got, K.causal_attn(q, k, v, slopes=slopes.double()))


# ---- one token -----------------------------------------------------------------------------------------------------
def decode(K, kind, g, b, h, hkv, ps, keys, lens, window, sinks, softcap, slopes, size=1.0):
    width = -(-keys // ps)
    pages = b * width + 1
    (kp, ks), (vp, vs) = pool_of(g, kind, hkv, pages, ps), pool_of(g, kind, hkv, pages, ps)
    p, q = table_of(g, b, width, pages), normal(g, b, h, D) * size
    if kind == "f16":
        got = K.page_flash_attn(p, q, kp, vp, pages * ps, b, width * ps, h, D, page_size=ps, seq_lens=lens, window=window, sinks=sinks, softcap=softcap, slopes=slopes)
    else:
        got = K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=ps, seq_lens=lens, window=window, sinks=sinks, softcap=softcap, slopes=slopes)
    t = torch.arange(width * ps, device="cuda")
    slots, n = p.long()[:, t // ps] * ps + t % ps, lens[:, None].long()
    seen, far = t[None] < n, (n - 1 - t[None]).clamp(min=0)
    if window:
        seen &= (far < window) | (t[None] < sinks)
    want, size, off = attention(q, values(kp, ks, ps)[:, slots], values(vp, vs, ps)[:, slots], seen, far, softcap, slopes)
    assert ((got.double() - want).abs() <= 2 ** -11 * want.abs() + WEIGHT * size + off + 2 ** -25).all()
    return got


LENS = [0, 1, 2, 15, 16, 17, 33, 64, 65, 129, 256, 300]


@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
@pytest.mark.parametrize("softcap,alibi", [(50.0, False), (0.5, False), (None, True), (20.0, True)])
@pytest.mark.parametrize("h,hkv,ps,window,sinks", [(4, 4, 16, None, 0), (4, 2, 16, 40, 4), (9, 3, 5, 64, 0), (8, 2, 64, 17, 33), (5, 1, 1, 100, 1), (18, 2, 16, None, 0), (8, 1, 20, 1, 0), (12, 1, 32, 300, 7)])
def test_token(K, kind, softcap, alibi, h, hkv, ps, window, sinks):
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    got = decode(K, kind, generator(h * ps), len(LENS), h, hkv, ps, 300, lens, window, sinks, softcap, slopes_of(h) if alibi else None)
    assert not got[0].any()


@pytest.mark.parametrize("kind", ["f16", "int8"])
@pytest.mark.parametrize("b,h,hkv,keys", [(1, 32, 32, 1), (1, 8, 1, 20001), (70, 32, 32, 700), (3, 32, 8, 9000), (200, 8, 8, 130)])
def test_token_long(K, kind, b, h, hkv, keys):
    g = generator(keys)
    lens = torch.randint(keys // 3, keys + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = keys
    decode(K, kind, g, b, h, hkv, 16, keys, lens, None, 0, 30.0, slopes_of(h))


def test_token_steep_and_large(K):
    g = generator(4)
    lens = torch.tensor([500, 77], dtype=torch.int32, device="cuda")
    decode(K, "f16", g, 2, 4, 4, 16, 500, lens, None, 0, None, torch.tensor([50.0, -2.0, 0.0, 1e-4], device="cuda"))
    for softcap in (0.01, 1.0, 1000.0):
        decode(K, "f16", g, 2, 4, 2, 16, 500, lens, None, 0, softcap, None, size=30.0)


# ---- calls ---------------------------------------------------------------------------------------------------------
def test_refusals(K):
    g = generator(1)
    q, k = normal(g, 20, 4, D), normal(g, 20, 2, D)
    int32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    one = torch.ones(4, device="cuda")
    for bad in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=math.nan), dict(softcap=1e4), dict(slopes=one[:3]), dict(slopes=one.int()), dict(slopes=one.cpu()),
                dict(documents=int32(0, 20).long()), dict(documents=int32(0, 20)[None]), dict(documents=int32()), dict(documents=int32(0, 20), offset=1), dict(prefix=-1),
                dict(prefix=int32(1)), dict(documents=int32(0, 20), prefix=int32(1, 2)), dict(documents=int32(0, 20), prefix=int32(1).long()), dict(documents=int32(0, 20).cpu()),
                dict(softcap=5.0, window=0), dict(softcap=5.0, sinks=-1), dict(softcap=5.0, offset=1), dict(softcap=5.0, offset=-1), dict(softcap=5.0, out=k),
                dict(softcap=5.0, out=q.float())):
        with pytest.raises(K.Q40Error):
            K.causal_attn(q, k, k, **bad)
    for bad in (q.float(), q[..., ::2], q.transpose(0, 1).contiguous().transpose(0, 1), q.cpu(), q[0]):
        with pytest.raises(K.Q40Error):
            K.causal_attn(bad, k, k, softcap=5.0)
    pool, p = normal(g, 2, 32, D), torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    for bad in (dict(softcap=0.0), dict(softcap=2000.0), dict(slopes=one[:1]), dict(slopes=one.cpu())):
        with pytest.raises(K.Q40Error):
            K.page_flash_attn(p, q[:3], pool, pool, 32, 3, 32, 4, D, page_size=16, **bad)
    assert K.causal_attn(q[:0], k, k, softcap=5.0).shape == (0, 4, D)
    assert K.page_flash_attn(p[:0], q[:0], pool, pool, 32, 0, 32, 4, D, page_size=16, softcap=5.0).shape == (0, 4, D)


def test_captured_on_another_stream_and_replayed(K):
    """With what the documents and lengths are when it is replayed; two graphs in turn, and beside eager calls."""
    g = generator(2)
    s, h = 500, 4
    q, k, v = normal(g, s, h, D), normal(g, s, h, D), normal(g, s, h, D)
    documents = torch.tensor([0, 100, 500], dtype=torch.int32, device="cuda")
    slopes, pool, p = slopes_of(h), normal(g, h, 512, D), torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
    lens = torch.tensor([10, 200], dtype=torch.int32, device="cuda")
    calls = [lambda: K.causal_attn(q, k, v, documents=documents, slopes=slopes, softcap=9.0),
             lambda: K.page_flash_attn(p, q[:2], pool, pool, 512, 2, 256, h, D, page_size=16, seq_lens=lens, softcap=9.0, slopes=slopes)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for call in calls:
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(call())
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    documents.copy_(torch.tensor([3, 290, 470], dtype=torch.int32))
    lens.copy_(torch.tensor([256, 3], dtype=torch.int32))
    for _ in range(2):
        for graph in graphs:
            graph.replay()
        for call, out in zip(calls, outs):
            assert torch.equal(call(), out)
