"""Prompts of more blocks than there are SMs, whose outputs go by way of shared memory, against the definition in 64 bits, for some of the heads."""
import math

import pytest
import torch
from test_gpu_pages import D, generator, normal
from test_gpu_scores import K, attention, check, mask, slopes_of  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

H, HKV, REP = 32, 8, 4
SIZES = [1281, 2049]                                      # 6 and 9 blocks a head


def int32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


def inputs(s, size=1.0):
    qkv = normal(generator(s), s, H + 2 * HKV, D)         # views of one projection's output
    qkv[:, :H] *= size
    return qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:]


def compare(got, q, k, v, seen, far, softcap=None, slopes=None):
    for g in (0, 5):
        heads = slice(g * REP, (g + 1) * REP)
        wide = lambda x: x[:, g:g + 1].double().transpose(0, 1)[:, None]
        check(got[:, heads], *attention(q[:, heads], wide(k), wide(v), seen, far, softcap, None if slopes is None else slopes[heads]), q.shape[0], v)


MASKS = [dict(), dict(documents=[0, 130, 700, 1281], prefixes=None), dict(documents=[300, 301, 900, 1200], prefixes=[5, 200, 1000]), dict(prefix=700), dict(window=300, sinks=5),
         dict(documents=[0, 513, 1000], window=100, sinks=140, prefix=90)]


@pytest.mark.parametrize("softcap,alibi,size", [(None, False, 1.0), (30.0, False, 1.0), (1.0, False, 8.0), (None, True, 1.0), (20.0, True, 4.0)])
@pytest.mark.parametrize("masks", MASKS)
@pytest.mark.parametrize("s", SIZES)
def test_large(K, s, masks, softcap, alibi, size):
    q, k, v = inputs(s, size)
    slopes = slopes_of(H) if alibi else None
    documents, prefixes, prefix, window, sinks = (masks.get(x) for x in ("documents", "prefixes", "prefix", "window", "sinks"))
    seen, far = mask(s, 0, window, sinks or 0, documents, prefixes, prefix or 0)
    call = dict(window=window, sinks=sinks or 0, softcap=softcap, slopes=slopes, documents=int32(documents), prefix=(prefix or 0) if prefixes is None else int32(prefixes))
    got = K.causal_attn(q, k, v, **call)
    assert K.tc_error_flag() == 0
    compare(got, q, k, v, seen, far, softcap, slopes)
    assert not got[~seen.any(1)].any()
    # rows of other strides: a multiple of 16 bytes, and not; what lies between them, and rows of no document, stay
    for ld in (H * D + 8, H * D + 2):
        room = torch.full((s * ld + 8,), 7.0, dtype=torch.float16, device="cuda")
        out = room.as_strided((s, H, D), (ld, D, 1), 0)
        assert K.causal_attn(q, k, v, out, **call) is out
        some = seen.any(1)
        assert torch.equal(out[some], got[some]) and (out[~some] == 7).all()
        assert (room.as_strided((s, ld - H * D), (ld, 1), H * D) == 7).all() and (room[s * ld:] == 7).all()


@pytest.mark.parametrize("softcap,alibi", [(None, False), (10.0, True)])
def test_values_that_are_not_finite(K, softcap, alibi):
    """In tiles that are seen whole, and in part; of infinities of both signs in one row, no number comes."""
    s, documents, prefixes = 1281, [0, 700, 1250], [150, 20]
    q, k, v = inputs(s)
    slopes = slopes_of(H) if alibi else None
    seen, far = mask(s, 0, None, 0, documents, prefixes)
    call = lambda: K.causal_attn(q, k, v, softcap=softcap, slopes=slopes, documents=int32(documents), prefix=int32(prefixes))
    plain = call()
    for j in (0, 149, 400, 699, 700, 1000, 1249, 1270):
        kept = v.clone()
        v[j, 0, 5], v[j, 5, 9], v[j, 5, 127] = math.inf, math.nan, -math.inf
        got = call()
        assert ((got[:, :REP, 5] == math.inf) == seen[:, j, None]).all() and (got[:, 5 * REP:6 * REP, 9].isnan() == seen[:, j, None]).all()
        assert ((got[:, 5 * REP:6 * REP, 127] == -math.inf) == seen[:, j, None]).all()
        same = torch.ones_like(got, dtype=torch.bool)
        same[:, :REP, 5], same[:, 5 * REP:6 * REP, 9], same[:, 5 * REP:6 * REP, 127] = False, False, False
        assert torch.equal(got[same], plain[same]) and K.tc_error_flag() == 0
        v.copy_(kept)
    v[10, 0, 5], v[300, 0, 5] = math.inf, -math.inf
    got = call()[:, :REP, 5]
    both, one = seen[:, 10] & seen[:, 300], seen[:, 10] & ~seen[:, 300]
    assert got[both].isnan().all() and (got[one] == math.inf).all() and got[~seen[:, 10] & ~seen[:, 300]].isfinite().all()


def test_keys_that_are_not_finite(K):
    """A score that is no number makes none of the rows that see it, and of no other."""
    s, documents = 1281, [100, 700, 1200]
    q, k, v = inputs(s)
    seen, _ = mask(s, 0, None, 0, documents)
    k[300], k[1250] = math.nan, math.nan
    for softcap in (None, 10.0):
        got = K.causal_attn(q, k, v, documents=int32(documents), softcap=softcap)
        assert (got[..., 0].isnan() == seen[:, 300, None]).all() and not got[~seen.any(1)].any()
