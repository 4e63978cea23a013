"""Append to a paged cache, attention over pages of fp16 or of 8 bits, and windows, each against its definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128
TYPES = {"f16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from spec_mcts_b200 import kernels
    return kernels


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").half()


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pool_of(g, kind, hkv, pages, ps):
    """Codes of every value a pool may hold and scales of unlike size (None for fp16)."""
    if kind == "f16":
        return normal(g, hkv, pages * ps, D), None
    if kind == "int8":
        codes = torch.randint(-127, 128, (hkv, pages * ps, D), generator=g, device="cuda").to(torch.int8)
    else:
        codes = (torch.randn((hkv, pages * ps, D), generator=g, device="cuda") * 120).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, torch.rand((hkv, pages), generator=g, device="cuda") * (3.0 / TOP[kind]) + 1e-4


def values(pool, scale, ps):
    return pool.double() if scale is None else pool.double() * scale.double().repeat_interleave(ps, 1)[..., None]


def table_of(g, b, width, pages, dtype=torch.int32):
    return torch.randperm(max(pages, b * width), generator=g, device="cuda")[:b * width].remainder(pages).view(b, width).to(dtype)


def attention(q, k, v, seen):
    """softmax over the seen keys of q [rows, H, D], k / v [Hkv, rows or 1, keys, D], seen [rows, keys]; and the same of |v|"""
    b, h, _ = q.shape
    hkv = k.shape[0]
    qh = q.double().view(b, hkv, h // hkv, D).transpose(0, 1)
    score = (qh @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(~seen[None, :, None], -math.inf)
    w = torch.softmax(score, -1).nan_to_num(0.0)
    clean = lambda x: x.masked_fill(~seen.any(0)[None, None, :, None], 0.0) if x.shape[1] == 1 else x.masked_fill(~seen[None, ..., None], 0.0)
    v = clean(v)
    back = lambda x: x.transpose(0, 1).reshape(b, h, D)
    return back(w @ v), back(w @ v.abs())


# A weight's relative error: its score is an fp32 sum over 128 products of up to 10 in all (in powers of two: 128 x 2^-24 x 10 x ln 2 = 5.3e-5), 2^x
# and log2 are approximate to 2^-22, weights in two parts to 2^-22; once in the sum of weights and once in that of values
WEIGHT = 2 * (5.3e-5 + 4 * 2 ** -22)


def check_decode(got, want, size):
    bound = 2 ** -11 * want.abs() + WEIGHT * size + 2 ** -25
    assert ((got.double() - want).abs() <= bound).all()


def decode(K, kind, g, b, h, hkv, ps, keys, lens, window, sinks, idx=torch.int32):
    width = -(-keys // ps)
    pages = b * width + 1
    (kp, ks), (vp, vs) = pool_of(g, kind, hkv, pages, ps), pool_of(g, kind, hkv, pages, ps)
    p, q = table_of(g, b, width, pages, idx), normal(g, b, h, D)
    t = torch.arange(width * ps, device="cuda")
    slots = p.long()[:, t // ps] * ps + t % ps
    n = lens[:, None].long()
    seen = t[None] < n
    if window:
        seen &= (n - 1 - t[None] < window) | (t[None] < sinks)
    want, size = attention(q, values(kp, ks, ps)[:, slots], values(vp, vs, ps)[:, slots], seen)
    if kind == "f16":
        run = lambda lens=lens: K.page_flash_attn(p, q, kp, vp, pages * ps, b, width * ps, h, D, page_size=ps, seq_lens=lens, window=window, sinks=sinks)
    else:
        run = lambda lens=lens: K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=ps, seq_lens=lens, window=window, sinks=sinks)
    return run, want, size, (p, q, kp, vp, ks, vs, seen, slots)


LENS = [0, 1, 2, 7, 8, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 200, 255, 256, 257, 300]


# heads of a kv head: 1, 2, 3, 4, 5, 8, 9 and 12 (two groups); pages that are and are not powers of two, longer than a tile, of one token
@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
@pytest.mark.parametrize("h,hkv,ps,window,sinks,idx", [(4, 4, 16, None, 0, torch.int32), (4, 2, 16, 40, 4, torch.int16), (9, 3, 5, 64, 0, torch.int32), (8, 2, 64, 17, 33, torch.int32),
                                                       (5, 1, 1, 100, 1, torch.int16), (16, 2, 20, 128, 16, torch.int32), (18, 2, 16, None, 0, torch.int32),
                                                       (12, 1, 32, 1, 0, torch.int32), (24, 3, 16, 1, 1, torch.int64), (2, 2, 300, 1000, 7, torch.int32)])
def test_decode_edges(K, kind, h, hkv, ps, window, sinks, idx):
    if kind == "f16" and window is None:
        window = 1 << 40                                  # all of them
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    run, want, size, _ = decode(K, kind, generator(h * ps), len(LENS), h, hkv, ps, 300, lens, window, sinks, idx)
    got = run()
    check_decode(got, want, size)
    assert not got[0].any()                               # no key at all
    assert torch.equal(run(), got)


# units of one and of several chunks in each of the rule's ranges
@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
@pytest.mark.parametrize("b,h,hkv,keys,window,sinks", [(1, 1, 1, 1, 4096, 0), (1, 8, 1, 20001, None, 0), (2, 32, 8, 3000, 2500, 4), (10, 32, 8, 1030, None, 0),
                                                       (17, 32, 32, 1500, 1100, 64), (70, 32, 32, 2100, None, 0), (1, 8, 8, 70000, None, 0),
                                                          (3, 32, 8, 40000, None, 0), (2, 16, 8, 129, 129, 0), (5, 8, 8, 1100, 1000, 30), (30, 16, 2, 3000, None, 0)])
def test_decode_long(K, kind, b, h, hkv, keys, window, sinks):
    if kind == "f16" and window is None:
        window, sinks = keys - 1, 1
    g = generator(keys)
    lens = torch.randint(keys // 3, keys + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = keys
    run, want, size, _ = decode(K, kind, g, b, h, hkv, 16, keys, lens, window, sinks)
    check_decode(run(), want, size)


@pytest.mark.parametrize("lens", [[18944, 18945, 37888, 37889], [75776, 75777, 76800, 76801], [511, 512, 513, 1]])
def test_decode_where_chunks_get_larger(K, lens):
    """Eight units: chunks double behind 37 of 512 and of 1024 keys, and are of 512 again behind 37 of 2048, up to 150 of them."""
    g = generator(lens[0])
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    run, want, size, _ = decode(K, "int8", g, 4, 4, 2, 64, max(lens), n, None, 0)
    check_decode(run(), want, size)


@pytest.mark.parametrize("kind", ["f16", "int8"])
def test_decode_does_not_depend_on_the_tables_width(K, kind):
    """Nor on what its entries behind the lengths are."""
    g = generator(5)
    lens = torch.tensor([700, 40, 0, 512], dtype=torch.int32, device="cuda")
    run, *_, (p, q, kp, vp, ks, vs, _, _) = decode(K, kind, g, 4, 8, 2, 16, 700, lens, 600, 3)
    wide = torch.full((4, 3 * p.shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda")
    for i in range(4):
        wide[i, :-(-int(lens[i]) // 16)] = p[i, :-(-int(lens[i]) // 16)]
    if kind == "f16":
        got = K.page_flash_attn(wide, q, kp, vp, kp.shape[1], 4, 16 * wide.shape[1], 8, D, page_size=16, seq_lens=lens, window=600, sinks=3)
    else:
        got = K.page_flash_attn_q8(wide, q, kp, vp, ks, vs, page_size=16, seq_lens=lens, window=600, sinks=3)
    assert torch.equal(got, run())


def test_decode_without_lengths_and_with_strides(K):
    g = generator(6)
    lens = torch.full((3,), 96, dtype=torch.int32, device="cuda")
    run, want, size, (p, q, kp, vp, ks, vs, _, _) = decode(K, "int8", g, 3, 4, 2, 16, 96, lens, None, 0)
    base = run()
    check_decode(base, want, size)
    assert torch.equal(run(lens=None), base)
    assert torch.equal(K.page_flash_attn_q8(p.repeat_interleave(2, 1)[:, ::2], torch.cat((q, q), 1)[:, :4], kp, vp, ks, vs, page_size=16), base)
    off = torch.empty(q.numel() + 1, dtype=torch.float16, device="cuda")[1:].view_as(q).copy_(q)
    assert torch.equal(K.page_flash_attn_q8(p, off, kp, vp, ks, vs, page_size=16), base)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("h", [2, 8])
def test_decode_masked_places_hold_anything(K, kind, h):
    """NaN and infinities in keys, values and scales that no query sees."""
    g = generator(7)
    lens = torch.tensor([90, 47, 0], dtype=torch.int32, device="cuda")
    run, want, size, (p, q, kp, vp, ks, vs, seen, slots) = decode(K, kind, g, 3, h, 1, 1, 96, lens, 20, 3)
    used = torch.zeros(kp.shape[1], dtype=torch.bool, device="cuda")
    used[slots[seen]] = True
    for pool, scale in ((kp, ks), (vp, vs)):
        if scale is None:
            pool[:, ~used] = float("nan")
        else:
            scale[:, ~used] = float("nan")
            pool.view(torch.uint8)[:, ~used] = 0x7f
    check_decode(run(), want, size)


@pytest.mark.parametrize("h", [2, 8])
@pytest.mark.parametrize("far", [9, 20, 40, 63, 600])     # in the same product, warp, CTA and another one
def test_decode_infinite_and_nan_values(K, h, far):
    """fp16: an infinite value comes out, whatever its weight is; 8 bits: a NaN scale does."""
    g = generator(8)
    n = 1000 if far > 63 else 64
    lens = torch.full((2,), n, dtype=torch.int32, device="cuda")
    run, *_, (p, q, kp, vp, ks, vs, _, slots) = decode(K, "f16", g, 2, h, 1, 16, n, lens, n, 0)
    q[..., 0] = 8.0
    kp[0, slots[0, 5], 0], kp[0, slots[0, far], 0] = -400.0, 40.0       # its score is far below another's
    vp[0, slots[0, 5], 3], vp[0, slots[0, 5], 70] = math.inf, -math.inf
    got = run()
    assert (got[0, :, 3] == math.inf).all() and (got[0, :, 70] == -math.inf).all() and got[0].isfinite().sum() == h * (D - 2) and got[1].isfinite().all()
    run, *_, (p, q, kp, vp, ks, vs, _, slots) = decode(K, "int8", g, 2, h, 1, 16, n, lens, None, 0)
    vs[0, p[1, 2].item()] = math.nan
    got = run()
    assert got[0].isfinite().all() and got[1].isnan().all()


def test_decode_scales_far_apart(K):
    """Pages of values 2^40 apart, of zeros, and of keys whose scale is 0."""
    g = generator(9)
    lens = torch.full((2,), 128, dtype=torch.int32, device="cuda")
    run, _, _, (p, q, kp, vp, ks, vs, seen, slots) = decode(K, "int8", g, 2, 4, 2, 16, 128, lens, None, 0)
    vs[:, ::3] *= 2.0 ** -40
    vs[:, 1::5] = 0.0
    ks[:, 2::5] = 0.0
    want, size = attention(q, values(kp, ks, 16)[:, slots], values(vp, vs, 16)[:, slots], seen)
    check_decode(run(), want, size)


# ---- prompts -------------------------------------------------------------------------------------------------------
def prompt_reference(q, k, v, window, sinks, offset):
    s = q.shape[0]
    i, j = torch.arange(offset, offset + s, device="cuda")[:, None], torch.arange(offset + s, device="cuda")[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    return attention(q, k[:offset + s].double().transpose(0, 1)[:, None], v[:offset + s].double().transpose(0, 1)[:, None], seen)


def check_prompt(got, want, size, v):
    # as in a decode step, and weights rounded to fp16: 2^-11 of each, or half a step of the smallest, 2^-25 of the largest weight
    bound = 2 ** -11 * want.abs() + (WEIGHT + 2 ** -11) * size + v.shape[0] * 2 ** -25 * v.float().nan_to_num(0, 0, 0).abs().max() + 2 ** -25
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("s,h,hkv,window,sinks,offset", [(1, 4, 4, 1, 0, 0), (1, 4, 2, 5, 2, 100), (16, 2, 1, 16, 0, 0), (63, 4, 2, 10, 1, 0), (64, 4, 2, 64, 64, 1), (65, 4, 1, 1, 0, 63),
                                                         (130, 8, 2, 40, 70, 200), (200, 2, 2, 1000, 5, 0), (200, 2, 2, 1000, 5, 777), (129, 3, 3, 128, 0, 128), (300, 4, 4, 65, 130, 450),
                                                         (77, 32, 8, 50, 4, 0), (257, 8, 1, 200, 4, 1000), (513, 16, 2, 1, 3, 0), (700, 5, 1, 333, 1000, 90),
                                                         (1000, 4, 2, 129, 0, 300), (1500, 2, 2, 700, 200, 31), (2049, 1, 1, 1, 1, 0), (1280, 2, 1, 10000, 0, 2000), (999, 2, 1, 128, 300, 129),
                                                         (1, 2, 1, 5000, 0, 4500), (7, 1, 1, 1000, 500, 6000), (100, 8, 2, 900, 4, 2000), (257, 4, 4, 300, 1, 3000), (300, 1, 1, 4000, 130, 3777)])
def test_prompt(K, s, h, hkv, window, sinks, offset):
    g = generator(s + h)
    q, k, v = normal(g, s, h, D), normal(g, offset + s + 3, hkv, D), normal(g, offset + s + 3, hkv, D)
    k[offset + s:], v[offset + s:] = math.nan, math.nan                  # rows behind the last position
    got = K.causal_attn(q, k, v, window=window, sinks=sinks, offset=offset)
    assert K.tc_error_flag() == 0
    check_prompt(got, *prompt_reference(q, k, v, window, sinks, offset), v)


def test_prompt_strided_into_out(K):
    g = generator(11)
    qkv, out = normal(g, 150, 8, D), torch.full((150, 6, D), 7.0, dtype=torch.float16, device="cuda")
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    got = K.causal_attn(q, k, v, out[:, 1:5], window=60, sinks=2)
    assert got.data_ptr() == out[:, 1:5].data_ptr()
    check_prompt(got, *prompt_reference(q, k, v, 60, 2, 0), v)
    assert (out[:, 0] == 7).all() and (out[:, 5] == 7).all()


@pytest.mark.parametrize("s,window", [(60, 30), (150, 30), (700, 30), (700, 650)])
def test_prompt_values_that_are_not_finite(K, s, window):
    """They reach the queries that see them, and no other; keys that are not finite reach nobody behind a mask."""
    g = generator(12)
    sinks = 3
    q, k, v = normal(g, s, 4, D), normal(g, s, 2, D), normal(g, s, 2, D)
    want, size = prompt_reference(q, k, v, window, sinks, 0)
    i = torch.arange(s, device="cuda")
    sees = lambda j: (i >= j) & ((i - j < window) | (j < sinks))
    x, y, z = s // 3, s // 3 + 20, s - 20
    v[x, 0, 5], v[x, 0, 6], v[y, 0, 6], v[z, 1, 7] = math.inf, math.inf, -math.inf, math.nan
    got = K.causal_attn(q, k, v, window=window, sinks=sinks)
    a, b, c = sees(x)[:, None], sees(y)[:, None], sees(z)[:, None]
    first, second = got[:, :2], got[:, 2:]
    assert ((first[..., 5] == math.inf) == a).all()
    assert ((first[..., 6] == math.inf) == (a & ~b)).all() and ((first[..., 6] == -math.inf) == (b & ~a)).all() and (first[..., 6].isnan() == (a & b)).all()
    assert (second[..., 7].isnan() == c).all()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[:, :2, 5:7], rest[:, 2:, 7] = False, False
    check_prompt(torch.where(rest, got, 0), torch.where(rest, want, 0), size, v)
    k[s // 2] = math.nan                                 # every query that sees it, and no other
    got = K.causal_attn(q, k, v, window=window, sinks=sinks)
    assert (got[..., 0].isnan() == sees(s // 2)[:, None]).all()


# ---- append --------------------------------------------------------------------------------------------------------
def tables(n):
    angle = torch.outer(torch.arange(n, device="cuda").double(), 1e4 ** (-torch.arange(64, device="cuda").double() / 64))
    return angle.cos().half(), angle.sin().half()


def rotated(x, at, cos, sin):
    """... and what the fp32 sum of its two products may be off"""
    c, s = cos[at].double()[:, None], sin[at].double()[:, None]
    a, b = x[..., :64].double(), x[..., 64:].double()
    off = (torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)) * 2 ** -24
    return torch.cat((a * c - b * s, b * c + a * s), -1), off


def check_fp16(got, want, off):
    assert ((got.double() - want).abs() <= 2 ** -11 * want.abs() + 2 * off + 2 ** -25).all()


def check_codes(kind, codes, want):
    """Codes of values that are `want` of a scale: half a step, and what fp32 quotients (two roundings, and the scale's two) may be off"""
    near = want.abs() * 2 ** -21
    half = torch.full_like(want, 0.5) if kind == "int8" else (want.abs() * 2 ** -4).clamp(min=2 ** -10)
    assert ((codes.double() - want).abs() <= half + near).all() and (codes.double().abs() <= TOP[kind]).all()


def append(K, kind, g, lens, starts, h, hkv, ps, rotate=True, decode_form=False, extra=0, idx=torch.int32):
    """One call, and each sequence's rows checked; everything else has to be as it was."""
    b, n_pos = len(lens), 400
    total = sum(lens) + extra
    width = max(1, max(-(-(s + n) // ps) for s, n in zip(starts, lens)))
    pages = b * width + 2
    (kp, ks), (vp, vs) = pool_of(g, kind, hkv, pages, ps), pool_of(g, kind, hkv, pages, ps)
    p = table_of(g, b, width, pages, idx)
    qkv = normal(g, total, h + 2 * hkv, D)
    qkv[:, h:] *= (0.1 + 3 * torch.rand((total, 1, 1), generator=g, device="cuda")).half()      # scales that grow, and that do not
    q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    cos, sin = tables(n_pos)
    offsets = torch.tensor([sum(lens[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
    pos = torch.tensor(starts, dtype=torch.int32, device="cuda")
    before = [None if x is None else x.clone() for x in (kp, vp, ks, vs)]
    got = K.page_append(p, k, v, kp, vp, pos, page_size=ps, offsets=None if decode_form else offsets, k_scale=ks, v_scale=vs,
                        **(dict(q=q, cos=cos, sin=sin) if rotate else {}))
    at = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)] + [torch.zeros(extra, dtype=torch.long)]).cuda().clamp(max=n_pos - 1)
    if rotate:
        want, off = rotated(q, at, cos, sin)
        check_fp16(got[:total - extra], want[:total - extra], off[:total - extra])
        assert not got[total - extra:].any()
    else:
        assert got is None
    for pool, scale, old_pool, old_scale, x, turn in ((kp, ks, before[0], before[2], k, rotate), (vp, vs, before[1], before[3], v, False)):
        want, off = rotated(x, at, cos, sin) if turn else (x.double(), torch.zeros_like(x, dtype=torch.float64))
        untouched = torch.ones(pages * ps, dtype=torch.bool, device="cuda")
        same_scale = torch.ones(pages, dtype=torch.bool, device="cuda")
        for i, (s, n) in enumerate(zip(starts, lens)):
            r, e = sum(lens[:i]), sum(lens[:i + 1])
            while r < e:                                  # a page at a time
                row, page = s % ps, int(p[i, s // ps]) & 0xffffffff
                m = min(ps - row, e - r)
                a = page * ps
                new, new_off = want[r:r + m].transpose(0, 1), off[r:r + m].transpose(0, 1)
                untouched[a + row:a + row + m] = False
                if kind == "f16":
                    check_fp16(pool[:, a + row:a + row + m], new, new_off) if turn else None
                    assert turn or torch.equal(pool[:, a + row:a + row + m], x[r:r + m].transpose(0, 1))
                else:
                    old = old_scale[:, page].double() if row else torch.zeros(hkv, dtype=torch.float64, device="cuda")
                    sc = torch.maximum(old, new.abs().amax((1, 2)) / TOP[kind])
                    assert ((scale[:, page].double() - sc).abs() <= 2 ** -22 * sc).all()
                    check_codes(kind, pool[:, a + row:a + row + m], new / sc[:, None, None])
                    held = old_pool[:, a:a + row]
                    grown = (scale[:, page] > old_scale[:, page])[:, None, None]
                    check_codes(kind, pool[:, a:a + row], torch.where(grown, held.double() * (old / sc)[:, None, None], held.double()))
                    assert torch.equal(torch.where(grown, held.view(torch.uint8), pool[:, a:a + row].view(torch.uint8)), held.view(torch.uint8))
                    untouched[a:a + row] = False
                    same_scale[page] = False
                r, s = r + m, s + m
        raw = lambda y: y.view(torch.uint8)
        assert torch.equal(raw(pool)[:, untouched], raw(old_pool)[:, untouched])
        assert scale is None or torch.equal(scale[:, same_scale], old_scale[:, same_scale])


@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
@pytest.mark.parametrize("starts,h,hkv,ps,idx", [([0], 4, 4, 16, torch.int32), ([0, 1, 7, 15, 16, 17, 31, 63, 100, 399, 450], 8, 2, 16, torch.int16), ([5, 0, 19, 20, 39], 3, 3, 20, torch.int32),
                                                 ([0, 3, 200], 6, 1, 1, torch.int32), ([0, 255, 256, 300], 32, 8, 256, torch.int64), (list(range(0, 300, 3)), 8, 8, 64, torch.int32)])
def test_append_one_token(K, kind, starts, h, hkv, ps, idx):
    append(K, kind, generator(len(starts)), [1] * len(starts), starts, h, hkv, ps, decode_form=True, idx=idx)


@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
@pytest.mark.parametrize("lens,starts,h,hkv,ps,extra", [([1], [0], 2, 2, 16, 0), ([40], [0], 2, 1, 16, 3), ([16, 0, 33, 1, 48], [0, 5, 15, 47, 16], 4, 2, 16, 0), ([100, 7], [3, 200], 8, 8, 20, 5),
                                                       ([130, 64, 65], [0, 63, 1], 3, 1, 64, 1), ([5, 9], [2, 0], 2, 2, 1, 0), ([300, 300], [0, 255], 4, 4, 256, 0), ([0, 0, 12, 0], [0, 3, 390, 9], 2, 1, 16, 2)])
@pytest.mark.parametrize("rotate", [True, False])
def test_append_runs(K, kind, lens, starts, h, hkv, ps, extra, rotate):
    append(K, kind, generator(sum(lens)), lens, starts, h, hkv, ps, rotate=rotate, extra=extra)


@pytest.mark.parametrize("kind", ["f16", "int8"])
def test_append_where_there_is_no_place(K, kind):
    """Positions below 0 and behind the table, and page ids out of the pool, are not written; the rest of the call is."""
    g = generator(13)
    hkv, ps, pages = 2, 16, 4
    (kp, ks), (vp, vs) = pool_of(g, kind, hkv, pages, ps), pool_of(g, kind, hkv, pages, ps)
    p = torch.tensor([[0], [1 << 30], [-1], [1], [2], [4]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([-1, 0, 0, 16, 0, 0], dtype=torch.int32, device="cuda")
    k, v = normal(g, 6, hkv, D), normal(g, 6, hkv, D)
    cos, sin = tables(32)
    q = normal(g, 6, 4, D)
    old = [x.clone() for x in (kp, vp)]
    got = K.page_append(p, k, v, kp, vp, pos, page_size=ps, k_scale=ks, v_scale=vs, q=q, cos=cos, sin=sin)
    for pool, o in zip((kp, vp), old):
        same = (pool.view(torch.uint8) == o.view(torch.uint8)).view(hkv, pages * ps, -1).all(-1)
        assert same.sum() == hkv * (pages * ps - 1) and not same[:, 2 * ps].any()
    assert not got[0].any() and torch.equal(got[4], q[4])
    # a run that begins below 0: its rows from position 0 on are there
    old = kp.clone()
    offsets = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    K.page_append(p[3:4], k, v, kp, vp, pos[:1] - 1, page_size=ps, offsets=offsets, k_scale=ks, v_scale=vs)
    same = (kp.view(torch.uint8) == old.view(torch.uint8)).view(hkv, pages * ps, -1).all(-1)
    assert not same[:, ps:ps + 4].any() and same.sum() == hkv * (pages * ps - 4)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_zeros_and_what_is_not_finite(K, kind):
    g = generator(14)
    (kp, ks), (vp, vs) = pool_of(g, kind, 1, 2, 16), pool_of(g, kind, 1, 2, 16)
    p, pos = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"), torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 1, D, dtype=torch.float16, device="cuda")
    v = normal(g, 2, 1, D)
    v[0, 0, 3], v[1, 0, 5] = math.inf, math.nan
    K.page_append(p, k, v, kp, vp, pos, page_size=16, k_scale=ks, v_scale=vs)
    assert not ks.any() and not kp[:, ::16].float().any() and vs.isnan().all()
    K.page_append(p, k, normal(g, 2, 1, D), kp, vp, pos + 1, page_size=16, k_scale=ks, v_scale=vs)
    assert vs.isnan().all()                              # until the pages are begun anew
    K.page_append(p, k, normal(g, 2, 1, D), kp, vp, pos, page_size=16, k_scale=ks, v_scale=vs)
    assert vs.isfinite().all()


@pytest.mark.parametrize("kind", ["f16", "int8", "e4m3"])
def test_a_chat_from_prompt_to_answer(K, kind):
    """Prompts by causal_attn and page_append, a later chunk of one behind them, then decode steps by page_append and paged attention: each output
    against attention over the whole sequence, as the cache holds it where the cache is read."""
    g = generator(15)
    h, hkv, ps, window, sinks, b, steps = 8, 2, 16, 40, 3, 2, 20
    cos, sin = tables(400)
    lens, width = [70, 33], 8
    p = table_of(g, b, width, b * width)
    dtype = TYPES[kind]
    zeros = lambda: torch.zeros(hkv, b * width * ps, D, device="cuda").to(dtype)
    scales = lambda: None if kind == "f16" else torch.zeros(hkv, b * width, device="cuda")
    kp, vp, ks, vs = zeros(), zeros(), scales(), scales()
    extra = dict(page_size=ps, k_scale=ks, v_scale=vs, cos=cos, sin=sin)
    x = normal(g, sum(lens), h + 2 * hkv, D)
    offsets = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device="cuda")
    K.page_append(p, x[:, h:h + hkv], x[:, h + hkv:], kp, vp, torch.zeros(b, dtype=torch.int32, device="cuda"), offsets=offsets, **extra)
    first = 0
    for n in lens:                                       # the prompts, in two chunks
        at = torch.arange(n, dtype=torch.int32, device="cuda")
        q, k, v = (y.clone() for y in (x[first:first + n, :h], x[first:first + n, h:h + hkv], x[first:first + n, h + hkv:]))
        K.rope_(q, at, cos, sin), K.rope_(k, at, cos, sin)
        got = torch.cat((K.causal_attn(q[:30], k, v, window=window, sinks=sinks), K.causal_attn(q[30:], k, v, window=window, sinks=sinks, offset=30)))
        check_prompt(got, *prompt_reference(q, k, v, window, sinks, 0), v)
        first += n
    now = torch.tensor(lens, dtype=torch.int32, device="cuda")
    t = torch.arange(width * ps, device="cuda")
    slots = p.long()[:, t // ps] * ps + t % ps
    for _ in range(steps):
        x = normal(g, b, h + 2 * hkv, D)
        q = K.page_append(p, x[:, h:h + hkv], x[:, h + hkv:], kp, vp, now, q=x[:, :h], **extra)
        now += 1
        seen = (t[None] < now[:, None]) & ((now[:, None] - 1 - t[None] < window) | (t[None] < sinks))
        want, size = attention(q, values(kp, ks, ps)[:, slots], values(vp, vs, ps)[:, slots], seen)
        if kind == "f16":
            got = K.page_flash_attn(p, q, kp, vp, kp.shape[1], b, width * ps, h, D, page_size=ps, seq_lens=now, window=window, sinks=sinks)
        else:
            got = K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=ps, seq_lens=now, window=window, sinks=sinks)
        check_decode(got, want, size)


def test_append_and_attention_in_a_graph_on_another_stream(K):
    """A captured step of two launches and their scratch, replayed: the positions it reads are on the device."""
    g = generator(16)
    b, h, hkv, ps, width = 3, 8, 2, 16, 40
    cos, sin = tables(700)
    p = table_of(g, b, width, b * width)
    (kp, ks), (vp, vs) = pool_of(g, "int8", hkv, b * width, ps), pool_of(g, "int8", hkv, b * width, ps)
    x, pos = normal(g, b, h + 2 * hkv, D), torch.tensor([500, 16, 300], dtype=torch.int32, device="cuda")
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")

    def step():
        q = K.page_append(p, x[:, h:h + hkv], x[:, h + hkv:], kp, vp, pos, page_size=ps, k_scale=ks, v_scale=vs, q=x[:, :h], cos=cos, sin=sin)
        lens.copy_(pos + 1)
        return K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=ps, seq_lens=lens)

    start = [y.clone() for y in (kp, vp, ks, vs)]
    eager = []
    for _ in range(3):
        eager.append(step())
        pos += 1
    eager_cache = [y.clone() for y in (kp, vp, ks, vs)]
    pos -= 3
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        for y, s in zip((kp, vp, ks, vs), start):
            y.view(torch.uint8).copy_(s.view(torch.uint8))
        for want in eager:
            graph.replay()
            assert torch.equal(out, want)
            pos += 1
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(y.view(torch.uint8), e.view(torch.uint8)) for y, e in zip((kp, vp, ks, vs), eager_cache))


def test_nothing_to_do(K):
    """No sequences, no tokens, tables without a page, queries of no position."""
    g = generator(18)
    (kp, ks), (vp, vs) = pool_of(g, "int8", 2, 4, 16), pool_of(g, "int8", 2, 4, 16)
    none = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")
    i32 = torch.int32
    assert K.page_flash_attn_q8(none(0, 2, dtype=i32), none(0, 4, D), kp, vp, ks, vs, page_size=16).shape == (0, 4, D)
    got = K.page_flash_attn_q8(none(2, 0, dtype=i32), normal(g, 2, 4, D), kp, vp, ks, vs, page_size=16)
    assert got.shape == (2, 4, D) and not got.any()
    before = [x.clone() for x in (kp, vp, ks, vs)]
    cos, sin = tables(8)
    extra = dict(page_size=16, k_scale=ks, v_scale=vs, cos=cos, sin=sin)
    assert K.page_append(none(0, 2, dtype=i32), none(0, 2, D), none(0, 2, D), kp, vp, none(0, dtype=i32), q=none(0, 4, D), **extra).shape == (0, 4, D)
    assert K.page_append(none(2, 2, dtype=i32), none(0, 2, D), none(0, 2, D), kp, vp, none(2, dtype=i32), offsets=none(3, dtype=i32), **extra) is None
    rows = normal(g, 3, 2, D)
    assert not K.page_append(none(0, 2, dtype=i32), rows, rows, kp, vp, none(0, dtype=i32), offsets=none(1, dtype=i32), q=normal(g, 3, 4, D), **extra).any()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((kp, vp, ks, vs), before))
    assert K.causal_attn(none(0, 4, D), normal(g, 7, 2, D), normal(g, 7, 2, D), window=3, offset=7).shape == (0, 4, D)


def test_split_calls_in_graphs_that_overlap(K):
    """Two captured graphs of calls with scratch, replayed at once on two streams, and eager calls on a third: each has scratch of its own."""
    g = generator(19)
    n = 6000
    q, k, v = normal(g, 60, 8, D), normal(g, n, 2, D), normal(g, n, 2, D)
    lens = torch.tensor([5000, 2000], dtype=torch.int32, device="cuda")
    run, *_ = decode(K, "e4m3", g, 2, 8, 2, 16, 5000, lens, None, 0)
    prompt = lambda: K.causal_attn(q, k, v, window=5000, sinks=4, offset=n - 60)
    want = [prompt(), run()]
    streams, graphs = [torch.cuda.Stream() for _ in range(3)], []
    for st in streams[:2]:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                out = [prompt(), run()]
            graphs.append((st, graph, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for st, graph, _ in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = [prompt(), run()]
    torch.cuda.synchronize()
    for outs in [o for *_, o in graphs] + [eager]:
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_calls_of_two_threads(K):
    import threading
    g = generator(20)
    lens = torch.tensor([3000, 1500, 700], dtype=torch.int32, device="cuda")
    run, *_ = decode(K, "int8", g, 3, 8, 2, 16, 3000, lens, None, 0)
    q, k, v = normal(g, 300, 4, D), normal(g, 2000, 2, D), normal(g, 2000, 2, D)
    prompt = lambda: K.causal_attn(q, k, v, window=1500, sinks=4, offset=1700)
    want, bad = [run(), prompt()], []

    def work(call, right):
        for _ in range(50):
            if not torch.equal(call(), right):
                bad.append(call)

    threads = [threading.Thread(target=work, args=a) for a in zip((run, prompt) * 2, want * 2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_without_the_extension(K, monkeypatch):
    """The general way of each call gives what the native one does."""
    g = generator(21)
    lens = torch.tensor([300, 17], dtype=torch.int32, device="cuda")
    calls = [decode(K, "int8", g, 2, 4, 2, 16, 300, lens, 100, 3)[0], decode(K, "f16", g, 2, 4, 2, 16, 300, lens, 100, 3)[0]]
    q, k, v = normal(g, 100, 4, D), normal(g, 100, 2, D), normal(g, 100, 2, D)
    calls.append(lambda: K.causal_attn(q, k, v, window=30))
    cos, sin = tables(64)
    p, pos = table_of(g, 2, 2, 4), torch.tensor([3, 16], dtype=torch.int32, device="cuda")
    start = [pool_of(g, "e4m3", 2, 4, 16) for _ in range(2)]

    def appended():
        (kp, ks), (vp, vs) = [(c.clone(), s.clone()) for c, s in start]
        versions = [x._version for x in (kp, ks, vp, vs)]
        out = K.page_append(p, k[:2], v[:2], kp, vp, pos, page_size=16, k_scale=ks, v_scale=vs, q=q[:2], cos=cos, sin=sin)
        assert all(x._version > n for x, n in zip((kp, ks, vp, vs), versions))      # the writes are counted
        return torch.cat([x.reshape(-1).float() for x in (out, kp, ks, vp, vs)])

    calls.append(appended)
    native = [c() for c in calls]
    monkeypatch.setattr(K, "_host_calls", None)
    assert all(torch.equal(c(), n) for c, n in zip(calls, native))


def test_refusals(K):
    g = generator(17)
    (kp, ks), (vp, vs) = pool_of(g, "int8", 2, 4, 16), pool_of(g, "int8", 2, 4, 16)
    p, q = table_of(g, 2, 2, 4), normal(g, 2, 4, D)
    k, v, pos = normal(g, 2, 2, D), normal(g, 2, 2, D), torch.zeros(2, dtype=torch.int32, device="cuda")
    ok = dict(page_size=16)
    bad = [lambda: K.page_flash_attn_q8(p, q, kp, vp, ks, None, **ok), lambda: K.page_flash_attn_q8(p, q, kp, vp, ks[:, :3], vs, **ok),
           lambda: K.page_flash_attn_q8(p, q, kp, vp, ks.half(), vs.half(), **ok), lambda: K.page_flash_attn_q8(p, q, kp.half(), vp.half(), ks, vs, **ok),
           lambda: K.page_flash_attn_q8(p, q, kp, vp.view(torch.float8_e4m3fn), ks, vs, **ok), lambda: K.page_flash_attn_q8(p, q, kp.transpose(0, 1), vp, ks, vs, **ok),
           lambda: K.page_flash_attn_q8(p, q.float(), kp, vp, ks, vs, **ok), lambda: K.page_flash_attn_q8(p[:1], q, kp, vp, ks, vs, **ok),
           lambda: K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=16, window=0), lambda: K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=16, window=4, sinks=-1),
           lambda: K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=15), lambda: K.page_flash_attn_q8(p, q[:, :3], kp, vp, ks, vs, **ok),
           lambda: K.page_flash_attn_q8(p, q, kp, vp, ks, vs, page_size=16, seq_lens=pos[:1]), lambda: K.page_flash_attn_q8(p.float(), q, kp, vp, ks, vs, **ok),
           lambda: K.page_flash_attn(p, q, kp.half(), vp.half(), 64, 2, 33, 4, D, page_size=16, window=4), lambda: K.page_flash_attn(p, q, kp.half(), vp.half(), 65, 2, 32, 4, D, page_size=16, window=4),
           lambda: K.page_flash_attn(p, q, kp, vp, 64, 2, 32, 4, D, page_size=16, window=4),
           lambda: K.page_append(p, k, v, kp, vp, pos, **ok), lambda: K.page_append(p, k, v, kp, vp, pos[:1], k_scale=ks, v_scale=vs, **ok),
           lambda: K.page_append(p, k[:, :1], v[:, :1], kp, vp, pos, k_scale=ks, v_scale=vs, **ok), lambda: K.page_append(p, k.float(), v, kp, vp, pos, k_scale=ks, v_scale=vs, **ok),
           lambda: K.page_append(p, k, v, kp, vp, pos, k_scale=ks, v_scale=vs, q=q, **ok), lambda: K.page_append(p, k, v, kp, vp, pos, k_scale=ks, v_scale=vs, offsets=pos, **ok),
           lambda: K.page_append(p, k, v, kp, vp, pos, k_scale=ks, v_scale=vs, cos=tables(4)[0], **ok), lambda: K.page_append(p, k, v, kp.half(), vp.half(), pos, k_scale=ks, v_scale=vs, **ok),
           lambda: K.page_append(p.cpu(), k, v, kp, vp, pos, k_scale=ks, v_scale=vs, **ok),
           lambda: K.causal_attn(q, q, q, window=0), lambda: K.page_flash_attn_q8(p.expand(2, 2).repeat(1, 1 << 17), q, kp, vp, ks, vs, page_size=1 << 30),
           lambda: K.causal_attn(q, q, q, window=3, sinks=-1), lambda: K.causal_attn(q, q, q, offset=1), lambda: K.causal_attn(q, q, q, offset=-1),
           lambda: K.causal_attn(q, q, q[:, :2], window=3), lambda: K.causal_attn(q, q[:, :3], q[:, :3], window=3), lambda: K.causal_attn(q, q, q, q[:1], window=3)]
    for call in bad:
        with pytest.raises(K.Q40Error):
            call()
