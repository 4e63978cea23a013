"""Calls of the paged cache and of windows that the other tests do not make, each against its definition in 64 bits."""
import math

import pytest
import torch

from test_gpu_pages import WEIGHT, D, K, append, check_decode, decode, generator, normal, prompt_reference  # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu
KINDS = ["f16", "int8", "e4m3"]


def general(q, k, v, window, sinks=0, offset=0, err=None, out=None):
    """The C call: without `err`, and without a workspace."""
    from spec_mcts_b200._lib import check, lib
    s, h, _ = q.shape
    o = torch.empty_like(q) if out is None else out
    check(lib.q40_attn_causal_window(q.data_ptr(), h * D, k.data_ptr(), k.shape[1] * D, v.data_ptr(), v.shape[1] * D, o.data_ptr(), o.stride(0), s, h, k.shape[1], D, offset, window,
                                     sinks, None, 0, None if err is None else err.data_ptr(), torch.cuda.current_stream().cuda_stream), "q40_attn_causal_window")
    return o


def check_weights(got, want, size, v):
    """Weights are off by 2^-11 of each, or, where that is more, by half a step of the smallest fp16 (2^-25) when a row's largest is at least 2^7; the rest
    as in a decode step, whose scores, powers and sums are off by `WEIGHT`."""
    bound = 2 ** -11 * want.abs() + (WEIGHT + 2 ** -11) * size + v.shape[0] * 2 ** -32 * v.float().nan_to_num(0, 0, 0).abs().max() + 2 ** -25
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("way", ["tensor cores", "general"])
@pytest.mark.parametrize("s,h,hkv,window,sinks,offset", [(300, 2, 1, 10000, 0, 8000), (1, 4, 2, 9000, 0, 8000), (300, 2, 2, 5000, 4, 8000), (17, 2, 2, 1000, 0, 100)])
def test_prompt_of_one_key_above_many(K, way, s, h, hkv, window, sinks, offset):
    """Weights 2^-26 of the first key's, whose value is 0: the result is what they sum up to."""
    g = generator(s + h)
    q, k, v = normal(g, s, h, D), torch.zeros(offset + s, hkv, D, dtype=torch.float16, device="cuda"), 1 + normal(g, offset + s, hkv, D) / 8
    q[..., 0] = 8.0
    k[0, :, 0] = 26 / (8 * 0.12751741)                # (1 / sqrt(128) log2 e)
    v[0] = 0
    run = K.causal_attn if way == "tensor cores" else lambda *a, **kw: general(*a, **kw)
    got = run(q, k, v, window=window, sinks=sinks, offset=offset)
    check_weights(got, *prompt_reference(q, k, v, window, sinks, offset), v)


@pytest.mark.parametrize("way", ["tensor cores", "general"])
@pytest.mark.parametrize("s,h,hkv,offset,far", [(700, 4, 2, 0, 300), (700, 4, 2, 0, 3), (60, 2, 1, 64, 70), (100, 8, 2, 2000, 1900), (300, 4, 4, 400, 500), (1, 2, 1, 3000, 2000)])
def test_prompt_infinite_values_of_keys_far_below(K, way, s, h, hkv, offset, far):
    """An infinite value comes out to every query that sees its key, whatever its weight is and whether or not all of a tile's queries see it."""
    g = generator(s + far)
    n = offset + s
    q, k, v = normal(g, s, h, D), normal(g, n, hkv, D), normal(g, n, hkv, D)
    q[..., 0] = 8.0
    k[5:7, :, 0], k[far, :, 0] = -400.0, 40.0         # scores far below the others, and one far above them
    late = n - 30 if s > 30 else n - 1                # in a tile that some queries see in part
    k[late, :, 0] = -400.0
    v[5, 0, 3], v[5, 0, 70], v[5:7, 0, 9], v[6, 0, 9], v[5, 0, 11], v[late, 0, 11], v[5, 0, 127] = torch.inf, -torch.inf, torch.inf, -torch.inf, torch.inf, -torch.inf, torch.nan
    run = K.causal_attn if way == "tensor cores" else lambda *a, **kw: general(*a, **kw)
    got = run(q, k, v, window=n, offset=offset)
    at = torch.arange(offset, n, device="cuda")[:, None]
    five, six, end = at >= 5, at >= 6, at >= late
    rep = got[:, :h // hkv]
    assert ((rep[..., 3] == torch.inf) == five).all() and ((rep[..., 70] == -torch.inf) == five).all() and (rep[..., 127].isnan() == five).all()
    assert ((rep[..., 9] == torch.inf) == (five & ~six)).all() and (rep[..., 9].isnan() == six).all()
    assert ((rep[..., 11] == torch.inf) == (five & ~end)).all() and (rep[..., 11].isnan() == end).all()
    clean = [x for x in range(D) if x not in (3, 9, 11, 70, 127)]
    assert rep[..., clean].isfinite().all() and got[:, h // hkv:].isfinite().all()
    fine = lambda x: torch.cat((x[:, :h // hkv, clean].flatten(1), x[:, h // hkv:].flatten(1)), 1)
    want, size = prompt_reference(q, k, v.nan_to_num(0, 0, 0), n, 0, offset)
    check_weights(fine(got), fine(want), fine(size), v)


def test_prompt_sum_of_many_weights(K):
    """The first key's value over the sum of 2^20 weights, each of which is 1.03 of a power of two: added one by one to a sum of 2^19 and more of that power, a weight would lose
    its 0.03.  Eighty heads, so that CTAs do not share the keys."""
    n, h = 1 << 20, 80
    q, k, v = (torch.zeros(s, dtype=torch.float16, device="cuda") for s in ((1, h, D), (n, 1, D), (n, 1, D)))
    q[..., 0], k[0, 0, 0], v[0] = 8.0, 9.9574 / (8 * 0.12751741), 1000.0
    got = K.causal_attn(q, k, v, window=n, offset=n - 1)
    assert K.tc_error_flag() == 0
    first = math.exp(8 * k[0, 0, 0].item() / math.sqrt(D))
    want = 1000 * first / (first + n - 1)
    # a weight's score, power and rounding (the first's value is exact); a step adds 128 weights to the sum, half a unit in the last place off: 2^-24 x 2^20 / 128
    assert (got.double() - want).abs().max() <= want * (2 ** -11 + WEIGHT + 2 ** -11 + 2 ** -11)


def test_decode_of_2_to_29_keys(K):
    """A table that lists one page over and over, and another one at the end of each sequence, with a key above all others: the last chunk of each unit."""
    g = generator(29)
    lens = [1 << 29, 65535 * 8192 + 1, 65535 * 8192]
    p = torch.zeros(3, 1 << 25, dtype=torch.int32, device="cuda")
    for i, n in enumerate(lens):
        p[i, (n - 1) // 16] = 1
    codes = torch.randint(-127, 128, (1, 32, D), generator=g, device="cuda").to(torch.int8)
    k, v, scale = codes.clone(), codes.clone(), torch.full((1, 2), 2.0 ** -7, device="cuda")
    k[..., 0] = -127
    k[0, [16 + (n - 1) % 16 for n in lens], 0] = 127          # 2^129 times the weight of the others, of which there are 2^29
    q = torch.zeros(3, 1, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 512.0
    q[..., 1:] = normal(g, 3, 1, D - 1) / 64
    got = K.page_flash_attn_q8(p, q, k, v, scale, scale, page_size=16, seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for i, n in enumerate(lens):
        seen = torch.arange(16, 16 + (n - 1) % 16 + 1, device="cuda")           # of the last page; the others do not count
        s = (k[0, seen].double() @ q[i, 0].double()) * 2.0 ** -7 / math.sqrt(D)
        want = torch.softmax(s, 0) @ (v[0, seen].double() * 2.0 ** -7)
        check_decode(got[i, 0], want, (v[0].double() * 2.0 ** -7).abs().amax().expand(D))


def test_page_sizes_that_no_call_takes(K):
    """Above 2^29: the native call refuses what the general way does."""
    g = generator(4)
    i32 = dict(dtype=torch.int32, device="cuda")
    p, pos, rows, q = torch.zeros(1, 1, **i32), torch.zeros(1, **i32), normal(g, 1, 2, D), normal(g, 1, 4, D)
    pool = torch.zeros(2, 64, D, dtype=torch.float16, device="cuda")
    for size in ((1 << 29) + 1, 1 << 30, 1 << 40):
        with pytest.raises(K.Q40Error):
            K.page_append(p, rows, rows, pool, pool.clone(), pos, page_size=size)
        with pytest.raises(K.Q40Error):
            K.page_flash_attn(p, q, pool, pool, 64, 1, 10, 4, D, page_size=size, window=4)
    assert not pool.any()


def test_prompt_behind_100_million_keys(K):
    """A CTA goes through its tiles for over a second: whoever waits for the last of them, or for all, does not give up after the 0.6 s of another wait.  One tensor of 26 GB is keys
    and values."""
    n, s, h = 100_000_000, 256, 148
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 30 GB")
    kv = torch.zeros(n, 1, D, dtype=torch.float16, device="cuda")
    q = torch.zeros(s, h, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0
    kv[n - 300, 0, 0] = kv[n - 10, 0, 0] = 100.0              # 2^102 times the weight of a key of zeros
    kv[n - 10, 0, 1] = 50.0
    got = K.causal_attn(q, kv, kv, window=n, offset=n - s)
    assert K.tc_error_flag() == 0
    want = torch.zeros_like(got)
    want[..., 0], want[s - 10:, :, 1] = 100.0, 25.0
    assert torch.equal(got, want)


# more than 148 units (sequences times groups of up to eight heads of a kv head), of one chunk of keys and of several: 2, 3, 4, 5, 7, 8 heads, and 12 as two groups
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("b,h,hkv,ps,keys,window,sinks", [(50, 8, 4, 16, 300, None, 0), (60, 9, 3, 20, 290, 200, 5), (100, 32, 8, 16, 520, None, 0), (160, 5, 1, 64, 130, 60, 0), (80, 14, 2, 16, 257, 100, 4),
                                                          (20, 64, 8, 64, 300, None, 0), (40, 24, 2, 16, 300, 256, 1), (80, 4, 2, 16, 1600, None, 0), (53, 12, 3, 16, 1500, 1400, 4),
                                                          (20, 64, 8, 16, 2000, None, 0), (170, 6, 1, 16, 1100, None, 0), (19, 64, 8, 64, 2300, 2100, 100)])
def test_decode_of_large_batches(K, kind, b, h, hkv, ps, keys, window, sinks):
    if kind == "f16" and window is None:
        window = keys
    g = generator(b + h + keys)
    lens = torch.randint(keys // 4, keys + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    lens[:4] = torch.tensor([keys, 0, 1, keys - 1])
    run, want, size, _ = decode(K, kind, g, b, h, hkv, ps, keys, lens, window, sinks)
    got = run()
    check_decode(got, want, size)
    assert not got[1].any() and torch.equal(run(), got)


# more than 32768 rows, where a lane group takes four heads: parts of fewer, and parts that go from keys to values (hkv 3, 5, 6, and 1 beside 5 heads)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("lens,starts,h,hkv,ps", [([1000, 0, 1, 777, 1100], [0, 5, 63, 100, 17], 6, 6, 64), ([4000, 1500], [3, 0], 5, 3, 100), ([9000, 7500], [0, 250], 1, 1, 256),
                                                  ([1201, 999, 1100], [15, 16, 17], 9, 5, 16)])
def test_append_of_long_runs(K, kind, rotate, lens, starts, h, hkv, ps):
    assert sum(lens) * ((h if rotate else 0) + 2 * hkv) > 32768
    append(K, kind, generator(sum(lens)), lens, starts, h, hkv, ps, rotate=rotate, extra=3)


@pytest.mark.parametrize("kind", KINDS)
def test_append_of_one_token_to_many_sequences(K, kind):
    append(K, kind, generator(3), [1] * 1500, [i % 391 for i in range(1500)], 14, 5, 64, decode_form=True)


@pytest.mark.parametrize("s,h,hkv,window,sinks,offset", [(1, 4, 2, 16, 4, 4000), (17, 4, 4, 16, 4, 4000), (64, 8, 2, 40, 10, 4001), (64, 2, 1, 1, 60, 999), (33, 3, 3, 20, 64, 700)])
def test_prompt_of_few_queries_far_from_the_first_keys(K, s, h, hkv, window, sinks, offset):
    g = generator(s)
    q, k, v = normal(g, s, h, D), normal(g, offset + s, hkv, D), normal(g, offset + s, hkv, D)
    check_weights(K.causal_attn(q, k, v, window=window, sinks=sinks, offset=offset), *prompt_reference(q, k, v, window, sinks, offset), v)


@pytest.mark.parametrize("s,h,hkv,window,sinks,offset", [(300, 4, 2, 100, 70, 500), (1, 2, 2, 3000, 0, 2900), (129, 8, 1, 33, 200, 0), (700, 2, 1, 10000, 0, 10)])
def test_prompt_by_the_general_kernel(K, s, h, hkv, window, sinks, offset):
    """No error word: the kernel for small calls, over several blocks of queries and many tiles."""
    g = generator(s)
    q, k, v = normal(g, s, h, D), normal(g, offset + s, hkv, D), normal(g, offset + s, hkv, D)
    check_weights(general(q, k, v, window, sinks, offset), *prompt_reference(q, k, v, window, sinks, offset), v)


@pytest.mark.parametrize("s,window,offset", [(100, 5000, 5000), (1, 4000, 4000), (257, 3000, 3000)])
def test_prompt_without_a_workspace(K, s, window, offset):
    """... CTAs do not share the keys."""
    g = generator(s)
    q, k, v = normal(g, s, 4, D), normal(g, offset + s, 2, D), normal(g, offset + s, 2, D)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    check_weights(general(q, k, v, window, 3, offset, err=err), *prompt_reference(q, k, v, window, 3, offset), v)
    assert not err.any()


@pytest.mark.parametrize("s", [60, 300])
@pytest.mark.parametrize("first,heads", [(2, 4), (0, 4), (8, 5)])
def test_prompt_into_rows_off_16_bytes(K, s, first, heads):
    """Output addresses that are multiples of 4 bytes, or rows that are not multiples of 16."""
    g = generator(s)
    q, k, v = normal(g, s, 4, D), normal(g, s, 2, D), normal(g, s, 2, D)
    ld = heads * D + (2 if heads == 5 else 0)
    room = torch.full((first + s * ld,), 7.0, dtype=torch.float16, device="cuda")
    out = room[first:].view(s, ld)[:, :4 * D].unflatten(1, (4, D))
    assert K.causal_attn(q, k, v, out, window=100, sinks=3).data_ptr() == out.data_ptr()
    check_weights(out, *prompt_reference(q, k, v, 100, 3, 0), v)
    assert (room[:first] == 7).all() and (room[first:].view(s, ld)[:, 4 * D:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
def test_a_prompt_in_chunks_as_documented(K, kind):
    """Two chunks: keys rotated by rope_ beside those that page_append puts in the cache, and, of fp16 pages, the cache's own."""
    from test_gpu_pages import TYPES, rotated, tables
    g = generator(40)
    total, done, h, hkv, ps, window, sinks = 200, 130, 8, 2, 16, 60, 3
    x, (cos, sin) = normal(g, total, h + 2 * hkv, D), tables(total)
    table = torch.randperm(13, generator=g, device="cuda", dtype=torch.int32)[None]
    kpool = torch.zeros(hkv, 13 * ps, D, device="cuda").to(TYPES[kind])
    vpool = kpool.clone()
    scales = {} if kind == "f16" else dict(k_scale=torch.zeros(hkv, 13, device="cuda"), v_scale=torch.zeros(hkv, 13, device="cuda"))
    k_of_one, v_of_one = (torch.zeros(total, hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    at = torch.arange(total, device="cuda")
    slots = table[0].long()[at // ps] * ps + at % ps
    for first, n in ((0, done), (done, total - done)):
        q, k, v = (y[first:first + n] for y in (x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]))
        q = K.page_append(table, k, v, kpool, vpool, torch.tensor([first], dtype=torch.int32, device="cuda"), page_size=ps, offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                          q=q, cos=cos, sin=sin, **scales)
        k_of_one[first:first + n].copy_(k), v_of_one[first:first + n].copy_(v)
        K.rope_(k_of_one[first:first + n], torch.arange(first, first + n, device="cuda"), cos, sin)
        # both products and their sum rounded by 2^-11 (2^13 times the 2^-24 of `products`), and 2^-25 where they are subnormal
        want, products = rotated(k, at[first:first + n], cos, sin)
        assert ((k_of_one[first:first + n].double() - want).abs() <= 8200 * products + 2 ** -11 * want.abs() + 3 * 2 ** -25).all()
        pairs = [(k_of_one, v_of_one)] + ([(p[:, slots].transpose(0, 1).contiguous() for p in (kpool, vpool))] if kind == "f16" else [])
        for ks, vs in pairs:
            got = K.causal_attn(q, ks, vs, window=window, sinks=sinks, offset=first)
            check_weights(got, *prompt_reference(q, ks, vs, window, sinks, first), vs)
