"""Operators of requests that share, fork and pack what they attend to, each one pass through its public entry point, and
the same in elementary torch operations.

  prompt   `causal_attn` with scores that are capped by a tanh or get a bias by distance, and with masks of documents (the
           prompts of several requests in one call) and of a prefix that sees itself in both directions.
  token    `page_flash_attn` and `page_flash_attn_q8` with such scores: one query for each sequence over its pages.
  fork     `page_fork`: sequences become continuations of others, whose pages they share, or are given up.
  extend   `page_extend`: sequences get the pages of their next tokens, and a copy of a page that they share and would write
           to; others give their last tokens back.
  compact  `page_compact`: pages in use move to the front of the pools.

Heads, head size and page sizes are those of the 7B and 70B architectures that the package is written for and of its tests;
the pools of `extend` and `compact` hold the pages of several layers side by side.
"""
from __future__ import annotations

import math

import torch

own = False

DEV, D = "cuda", 128
QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"f16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # a short question, of which the instructions in front see each other in both directions; capped scores
        {"name": "prompt_77", "kind": "prompt", "tokens": 77, "docs": 0, "prefix": 30, "softcap": 50.0, "alibi": False, "window": 0, "heads": 32, "kv_heads": 32},
        # the prompts of nine requests in one call, scores by distance
        {"name": "prompt_docs", "kind": "prompt", "tokens": 4001, "docs": 9, "prefix": 0, "softcap": 0.0, "alibi": True, "window": 0, "heads": 32, "kv_heads": 32},
        # a long prompt of the 70B geometry, capped scores, a layer that sees 4096 keys back
        {"name": "prompt_16384", "kind": "prompt", "tokens": 16384, "docs": 0, "prefix": 0, "softcap": 30.0, "alibi": False, "window": 4096, "heads": 64, "kv_heads": 8},
        # a short answer of one sequence
        {"name": "token_1", "kind": "token", "cache": "f16", "seqs": 1, "keys": 512, "softcap": 50.0, "alibi": False, "heads": 32, "kv_heads": 32, "page": 16, "window": 0},
        # a full batch, lengths anywhere up to the longest, scores by distance
        {"name": "token_64_e4m3", "kind": "token", "cache": "e4m3", "seqs": 64, "keys": 2048, "softcap": 0.0, "alibi": True, "heads": 32, "kv_heads": 32, "page": 16, "window": 0},
        # few very long sequences, eight query heads on each kv head, capped scores
        {"name": "token_long_int8", "kind": "token", "cache": "int8", "seqs": 8, "keys": 65536, "softcap": 30.0, "alibi": False, "heads": 64, "kv_heads": 8, "page": 64, "window": 0},
        # the branches of one search step behind a short prompt
        {"name": "fork_16", "kind": "fork", "seqs": 16, "keys": 500, "page": 16, "spare": 50},
        # a server's many sequences, some long, of which half go on as others
        {"name": "fork_512", "kind": "fork", "seqs": 512, "keys": 8000, "page": 16, "spare": 0},
        # the next token of ten branches, half of them just forked, in one layer's pools
        {"name": "extend_10", "kind": "extend", "cache": "f16", "seqs": 10, "keys": 600, "page": 16, "layers": 1, "kv_heads": 8, "spare": 10},
        # ... of a hundred, in the pools of sixteen layers
        {"name": "extend_100", "kind": "extend", "cache": "f16", "seqs": 100, "keys": 200, "page": 16, "layers": 16, "kv_heads": 8, "spare": 0},
        # one layer's pools after a few sequences have ended
        {"name": "compact_8", "kind": "compact", "cache": "f16", "seqs": 8, "keys": 400, "page": 16, "layers": 1, "kv_heads": 8, "spare": 50},
        # the pools of eight layers, more than half of whose pages are free, in 8 bits
        {"name": "compact_64_e4m3", "kind": "compact", "cache": "e4m3", "seqs": 64, "keys": 1000, "page": 16, "layers": 8, "kv_heads": 8, "spare": 200},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "token", "token", "fork", "extend", "compact"])
    heads, kv = rng.choice([(32, 32), (32, 8), (64, 8), (8, 1), (24, 6)])
    if kind in ("prompt", "token"):
        scores = rng.choice(["cap", "alibi", "both", "none" if kind == "prompt" else "cap"])
        case = {"kind": kind, "heads": heads, "kv_heads": kv, "softcap": round(_log(rng, 5, 100) * 1.0, 1) if scores in ("cap", "both") else 0.0,
                "alibi": scores in ("alibi", "both"), "window": rng.choice([0, 0, _log(rng, 1, 8192)])}
        if kind == "prompt":
            tokens = _log(rng, 1, 6000)
            docs = rng.choice([0, min(tokens, _log(rng, 1, 40))])
            return case | {"tokens": tokens, "docs": docs, "prefix": rng.choice([0, rng.randint(0, tokens)])}
        keys = _log(rng, 1, 32768)
        return case | {"cache": rng.choice(list(DTYPES)), "page": rng.choice([1, 16, 16, 20, 32, 64]), "keys": keys,
                       "seqs": min(_log(rng, 1, 128), max(1, 8 * 32768 * 8 // (keys * kv)))}
    page = rng.choice([1, 16, 16, 20, 32, 64])
    if kind == "fork":
        return {"kind": kind, "seqs": _log(rng, 1, 500), "keys": _log(rng, 1, 8000), "page": max(page, 4), "spare": _log(rng, 1, 5000)}
    case = {"kind": kind, "cache": rng.choice(["f16", "e4m3"]), "page": page, "seqs": _log(rng, 1, 128), "layers": rng.choice([1, 1, 2, 8]), "kv_heads": rng.choice([1, 4, 8])}
    pages = 200_000 // (page * case["layers"] * case["kv_heads"])                  # of 128 MB in all, at most
    keys = max(1, min(_log(rng, 1, 1500), pages * page // case["seqs"]))
    return case | {"keys": keys, "spare": rng.randint(1, max(1, pages // 2))}


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)


def _pool(gen, kind, heads, pages, page):
    """Pool and scales (None in fp16) of keys or values of usual size, channels of unlike size among them."""
    x = _normal(gen, heads, pages * page, D) * (0.5 + torch.rand((heads, 1, D), generator=gen, device=DEV)).half()
    if kind == "f16":
        return x, None
    x = x.view(heads, pages, page, D)
    scale = x.abs().amax((2, 3)).float() / QMAX[kind]
    y = x.float() / scale[..., None, None]
    codes = y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return codes.view(heads, -1, D), scale


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _slopes(heads):
    """Falling from head to head, as models with such a bias have them."""
    return torch.pow(2.0, -8.0 * torch.arange(1, heads + 1, dtype=torch.float64) / heads).float().to(DEV)


def _sizes(case):
    """Pages of the pools, which have room for all that no fork shares, and pages of a sequence at most."""
    most = -(-case["keys"] // case["page"])
    return sum(not (i % 4 and i % 2) for i in range(case["seqs"])) * most + case["spare"], most + most // 16 + 9


def _sequences(case, gen, host):
    """Table, lengths and references of sequences in groups of four: half of them as they came out of a fork of their group's first,
    the others with pages of their own behind a part that they share with it."""
    b, ps = case["seqs"], case["page"]
    ints = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=host).tolist()
    lens, share, fresh = ints((case["keys"] + 1) // 2, case["keys"], b), ints(0, case["keys"] // ps, b), [i % 4 and i % 2 for i in range(b)]
    rows, used = [], 0
    for i in range(b):
        first = i - i % 4
        if fresh[i]:
            lens[i] = lens[first]
            rows.append(rows[first])
            continue
        need = -(-lens[i] // ps)
        s = 0 if i == first else min(share[i], lens[first] // ps, need)
        rows.append((rows[first][:s] if s else []) + list(range(used, used + need - s)))
        used += need - s
    n_pages, width = _sizes(case)
    at = torch.full((b, width), -1, dtype=torch.int64)
    for i, r in enumerate(rows):
        at[i, :len(r)] = torch.tensor(r, dtype=torch.int64)
    at = at.to(DEV)
    # what lies behind a sequence's pages is left over from earlier ones
    ids = torch.randperm(n_pages, generator=gen, device=DEV)
    table = torch.where(at >= 0, ids[at.clamp(min=0)], torch.randint(0, n_pages, at.shape, generator=gen, device=DEV))
    refs = torch.zeros(n_pages, dtype=torch.int64, device=DEV).index_add_(0, table[at >= 0], torch.ones_like(table[at >= 0]))
    return table.int(), _int32(lens), refs.int(), n_pages


def prepare(case, seed):
    gen, host = torch.Generator(device=DEV).manual_seed(int(seed)), torch.Generator().manual_seed(int(seed))
    ints = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=host).tolist()
    st = dict(case)
    if case["kind"] == "prompt":
        n, h, hkv, docs = case["tokens"], case["heads"], case["kv_heads"], case["docs"]
        qkv = _normal(gen, n, h + 2 * hkv, D)            # one projection's output: its queries, keys and values are views
        st |= {"q": qkv[:, :h], "k": qkv[:, h:h + hkv], "v": qkv[:, h + hkv:], "slopes": _slopes(h) if case["alibi"] else None, "documents": None, "prefixes": None}
        if docs:
            cuts = sorted((torch.randperm(n - 1, generator=host)[:docs - 1] + 1).tolist()) if n > 1 else []
            st["documents"] = _int32([0] + cuts + [n])
            if case["prefix"]:
                st["prefixes"] = _int32(ints(0, case["prefix"], len(cuts) + 1))
        return st
    ps = case["page"]
    if case["kind"] == "token":
        b, h, hkv = case["seqs"], case["heads"], case["kv_heads"]
        lens = [case["keys"]] + ints(case["keys"] // 2, case["keys"], b - 1)
        width, pages = -(-case["keys"] // ps), b * -(-case["keys"] // ps)
        table = torch.randperm(pages, generator=gen, device=DEV).view(b, width).int()
        st |= {"q": _normal(gen, b, h, D), "lens": _int32(lens), "table": table, "slopes": _slopes(h) if case["alibi"] else None}
        (st["kpool"], st["kscale"]), (st["vpool"], st["vscale"]) = _pool(gen, case["cache"], hkv, pages, ps), _pool(gen, case["cache"], hkv, pages, ps)
        return st
    st["table"], st["lens"], st["refs"], n = _sequences(case, gen, host)
    b = case["seqs"]
    if case["kind"] == "fork":                           # half go on as they are, one in eight is given up, the others go on as any
        st["parents"] = _int32([i if x < 4 else -1 if x == 4 else y for i, (x, y) in enumerate(zip(ints(0, 7, b), ints(0, b - 1, b)))])
        return st
    heads = case["layers"] * case["kv_heads"]
    (st["kpool"], st["kscale"]), (st["vpool"], st["vscale"]) = _pool(gen, case["cache"], heads, n, ps), _pool(gen, case["cache"], heads, n, ps)
    if case["kind"] == "extend":                         # mostly a token; drafts of a few, and what is taken back of others
        st["add"] = _int32([1 if x < 12 else 0 if x == 12 else y if x < 15 else -y for x, y in zip(ints(0, 15, b), ints(2, 8, b))])
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _changed(score, st, far, head_dim):
    """Scores [.., heads.., queries, keys] capped, and less what the distances cost; slopes lie along `head_dim` dims from the end."""
    if st["softcap"]:
        score = torch.tanh(score / st["softcap"]) * st["softcap"]
    if st["slopes"] is not None:
        score = score - st["slopes"].view(*st["slope_shape"]) * far
    return score


def _prompt_plain(st, block=512):
    (n, h, _), w = st["q"].shape, st["window"] or st["tokens"]
    hkv, out, j = st["k"].shape[1], torch.empty((n, h, D), dtype=torch.float16, device=DEV), torch.arange(n, device=DEV)
    if st["documents"] is None:
        start, end, prefix = torch.zeros_like(j), torch.full_like(j, n), torch.full_like(j, st["prefix"])
    else:
        doc = torch.searchsorted(st["documents"][1:].contiguous(), j.int(), right=True)
        start, end = st["documents"][doc].long(), st["documents"][doc + 1].long()
        prefix = st["prefixes"][doc].long() if st["prefixes"] is not None else torch.zeros_like(j)
    st = st | {"slope_shape": (hkv, h // hkv, 1, 1)}
    for a in range(0, n, block):
        i, s, e, f = (x[a:a + block, None] for x in (j, start, end, start + prefix))
        lo, hi = max(0, a - w + 1) if st["documents"] is None else 0, n if st["prefix"] else min(n, a + block)
        key = j[None, lo:hi]
        seen = (key >= s) & (key < e) & ((key <= i) | (key < f)) & (i - key < w)
        k, v = (x[lo:hi].float().permute(1, 2, 0) for x in (st["k"], st["v"]))                       # [kv heads, D, keys]
        q = st["q"][a:a + block].float().view(i.shape[0], hkv, -1, D).permute(1, 2, 0, 3)            # [kv heads, heads of one, queries, D]
        score = _changed(q @ k[:, None] / math.sqrt(D), st, (i - key).abs(), 3).masked_fill(~seen, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        out[a:a + block] = (p @ v.transpose(1, 2)[:, None] / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).reshape(i.shape[0], h, D).half()
    return out


def _token_plain(st):
    ps, (b, h, _), n = st["page"], st["q"].shape, st["lens"][:, None].long()
    lo = (n - (st["window"] or st["keys"])).clamp(min=0)
    t = lo + torch.arange(min(st["keys"], st["window"] or st["keys"]), device=DEV)[None]
    there = t < n
    far = n - 1 - t
    t = torch.where(there, t, 0)
    slots = st["table"].gather(1, t // ps).long() * ps + t % ps
    k, v = (x[:, slots].float() if s is None else x.view(torch.uint8)[:, slots].view(x.dtype).float() * s[:, slots // ps][..., None]
            for x, s in ((st["kpool"], st["kscale"]), (st["vpool"], st["vscale"])))                  # [kv heads, sequences, keys, D]
    hkv = k.shape[0]
    q = st["q"].float().view(b, hkv, -1, D).transpose(0, 1)
    score = _changed(q @ k.transpose(-1, -2) / math.sqrt(D), st | {"slope_shape": (hkv, 1, h // hkv, 1)}, far[:, None], 3).masked_fill(~there[:, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))                             # a sequence without keys: zeros
    return (e @ v / e.sum(-1, keepdim=True).clamp(min=1e-30)).transpose(0, 1).reshape(b, h, D).half()


def _listed_pages(table, lens, ps):
    return torch.arange(table.shape[1], device=DEV)[None] < ((lens + ps - 1) // ps)[:, None]


def _fork_plain(st):
    table, lens, refs, parents, ps = st["table"], st["lens"], st["refs"], st["parents"].long(), st["page"]
    there, at = parents >= 0, parents.clamp(min=0)
    new_lens = torch.where(there, lens[at], 0)
    old, new = _listed_pages(table, lens, ps), _listed_pages(table, new_lens, ps)
    new_table = torch.where(new, table[at], 0)
    count = lambda t, m: torch.zeros(refs.shape[0] + 1, dtype=torch.int32, device=DEV).index_add_(
        0, torch.where(m, t, refs.shape[0]).flatten().long(), torch.ones(t.numel(), dtype=torch.int32, device=DEV))[:-1]
    return {"table": new_table, "lens": new_lens, "refs": refs + count(new_table, new) - count(table, old)}


def _move(st, src, dst, rows):
    """The first `rows` rows (a number for each) of pages src to pages dst of the pools."""
    ps = st["page"]
    for pool, scale in ((st["kpool"], st["kscale"]), (st["vpool"], st["vscale"])):
        x = pool.view(torch.uint8 if scale is not None else pool.dtype).view(pool.shape[0], -1, ps, D)
        keep = torch.arange(ps, device=DEV)[None, :, None] < rows[:, None, None]
        x[:, dst] = torch.where(keep, x[:, src], x[:, dst])
        if scale is not None:
            scale[:, dst] = scale[:, src]


def _extend_plain(st):
    table, refs, ps, (b, width), n_pages = st["table"], st["refs"].long(), st["page"], st["table"].shape, st["refs"].shape[0]
    n, add, row = st["lens"].long(), st["add"].long(), torch.arange(st["table"].shape[0], device=DEV)
    m = (n + add).clamp(min=0)
    n0, n1 = (n + ps - 1) // ps, (m + ps - 1) // ps
    grows = (add > 0) & (n1 <= width)
    tail = table.gather(1, (n // ps).clamp(max=width - 1)[:, None])[:, 0].long()
    partial = grows & (n % ps != 0)
    sink = torch.where(partial, tail, n_pages)
    writers = torch.zeros(n_pages + 1, dtype=torch.int64, device=DEV).index_add_(0, sink, torch.ones_like(sink))
    last = torch.full((n_pages + 1,), -1, dtype=torch.int64, device=DEV).scatter_reduce(0, sink, row, "amax")
    shared = refs[tail]
    copies = partial & (shared > 1) & ~((writers[tail] == shared) & (last[tail] == row))
    need = torch.where(grows, n1 - n0 + copies, 0)
    base = need.cumsum(0) - need
    free = (refs <= 0).nonzero()[:, 0]
    granted = grows & ((need == 0) | (base + need <= free.shape[0]))
    m, copies = torch.where(granted | (add <= 0), m, n), copies & granted
    n1 = (m + ps - 1) // ps
    j = torch.arange(width, device=DEV)[None]
    old, new = j < n0[:, None], j < n1[:, None]
    rank = base[:, None] + torch.where(j == (n0 - copies.long())[:, None], 0, j - (n0 - copies.long())[:, None])
    taken = new & (~old | (copies[:, None] & (j == n0[:, None] - 1)))
    given = torch.where(taken, torch.cat((free, free.new_zeros(1)))[torch.where(taken, rank, -1)], 0)
    new_table = torch.where(taken, given, torch.where(new, table.long(), 0))
    dropped = old & ~new
    refs = torch.cat((refs, refs.new_zeros(1)))
    refs = refs.index_add(0, torch.where(dropped, table.long(), n_pages).flatten(), -torch.ones(b * width, dtype=torch.int64, device=DEV))
    refs = refs.index_add(0, torch.where(copies, tail, n_pages), -torch.ones_like(tail))[:-1]
    refs[given[taken]] = 1
    src, dst = tail[copies], given.gather(1, (n // ps).clamp(max=width - 1)[:, None])[:, 0][copies]
    _move(st, src, dst, (n % ps)[copies])
    return {"table": new_table.int(), "lens": m.int(), "refs": refs.int(), **_pools_out(st)}


def _compact_plain(st):
    table, refs, ps = st["table"], st["refs"], st["page"]
    used, ids = refs > 0, torch.arange(refs.shape[0], device=DEV)
    front = ids < used.sum()
    src, dst = (used & ~front).nonzero()[:, 0], (~used & front).nonzero()[:, 0]
    where = torch.where(used, ids, -1)
    where[src] = dst
    _move(st, src, dst, torch.full_like(src, ps))
    new_refs = torch.where(front, refs, 0)
    new_refs[dst] = refs[src]
    listed_pages = _listed_pages(table, st["lens"], ps)
    new_table = torch.where(listed_pages, where[torch.where(listed_pages, table, 0).long()], 0)
    return {"table": new_table.int(), "refs": new_refs, "where": where.int(), **_pools_out(st)}


def _pools_out(st):
    return {"k": st["kpool"], "v": st["vpool"], "k_scale": st["kscale"], "v_scale": st["vscale"]}


def run(st):
    kind = st["kind"]
    if not own:
        return {"prompt": _prompt_plain, "token": _token_plain, "fork": _fork_plain, "extend": _extend_plain, "compact": _compact_plain}[kind](st)
    from spec_mcts_b200 import kernels as K
    if kind == "prompt":
        return K.causal_attn(st["q"], st["k"], st["v"], window=st["window"] or None, softcap=st["softcap"] or None, slopes=st["slopes"],
                             documents=st["documents"], prefix=st["prefix"] if st["documents"] is None else st["prefixes"])
    if kind == "token":
        scores = {"window": st["window"] or None, "softcap": st["softcap"] or None, "slopes": st["slopes"]}
        if st["cache"] != "f16":
            return K.page_flash_attn_q8(st["table"], st["q"], st["kpool"], st["vpool"], st["kscale"], st["vscale"], page_size=st["page"],
                                        seq_lens=st["lens"], **scores)
        b, h, _ = st["q"].shape
        return K.page_flash_attn(st["table"], st["q"], st["kpool"], st["vpool"], st["kpool"].shape[1], b, st["keys"], h, D, page_size=st["page"],
                                 seq_lens=st["lens"], **scores)
    if kind == "fork":
        table, lens, refs = K.page_fork(st["table"], st["lens"], st["refs"], st["parents"], page_size=st["page"])
        return {"table": table, "lens": lens, "refs": refs}
    if kind == "extend":
        table, lens, refs = K.page_extend(st["table"], st["lens"], st["refs"], st["kpool"], st["vpool"], st["add"], page_size=st["page"],
                                          k_scale=st["kscale"], v_scale=st["vscale"])
        return {"table": table, "lens": lens, "refs": refs, **_pools_out(st)}
    table, refs, where = K.page_compact(st["table"], st["lens"], st["refs"], st["kpool"], st["vpool"], page_size=st["page"],
                                        k_scale=st["kscale"], v_scale=st["vscale"])
    return {"table": table, "refs": refs, "where": where, **_pools_out(st)}


# ---- in 64 bits, head by head and sequence by sequence -------------------------------------------------------------
def _attend(q, k, v, softcap, cost, seen):
    """Attention of q [heads, rows, D] over k / v [keys, D], cost [heads, 1 or rows, keys] off the capped scores, or None."""
    score = torch.matmul(q, k.t()).mul_(1 / math.sqrt(D))
    if softcap:
        score = score.div_(softcap).tanh_().mul_(softcap)
    if cost is not None:
        score = score.sub_(cost)
    if seen is not None:
        score = score.masked_fill_(~seen, -math.inf)
    return torch.softmax(score, -1) @ v


def _exact_prompt(st, step=1024):
    n, h, hkv, w = st["tokens"], st["heads"], st["kv_heads"], st["window"] or st["tokens"]
    out = torch.empty((n, h, D), dtype=torch.float64, device=DEV)
    ends = [0, n] if st["documents"] is None else st["documents"].tolist()
    prefixes = [st["prefix"]] if st["documents"] is None else st["prefixes"].tolist() if st["prefixes"] is not None else [0] * (len(ends) - 1)
    slopes = None if st["slopes"] is None else st["slopes"].double().view(hkv, -1)
    for s, e, pre in zip(ends, ends[1:], prefixes):
        for g in range(hkv):
            heads = slice(g * (h // hkv), (g + 1) * (h // hkv))
            k, v = st["k"][s:e, g].double(), st["v"][s:e, g].double()
            for a in range(0, e - s, step):
                i = torch.arange(a, min(a + step, e - s), device=DEV)[:, None]
                lo, hi = max(0, a - w + 1), min(e - s, max(int(i[-1]) + 1, pre))
                j = torch.arange(lo, hi, device=DEV)[None]
                seen = torch.maximum(i, torch.full_like(i, pre - 1)) >= j
                seen &= j > i - w
                cost = None if slopes is None else slopes[g][:, None, None] * (i - j).abs()
                out[s + a:s + a + i.shape[0], heads] = _attend(st["q"][s + a:s + a + i.shape[0], heads].double().transpose(0, 1), k[lo:hi], v[lo:hi],
                                                               st["softcap"], cost, seen).transpose(0, 1)
    return out


def _exact_token(st):
    h, hkv, ps = st["heads"], st["kv_heads"], st["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    slopes = None if st["slopes"] is None else st["slopes"].double().view(hkv, -1)
    for b, n in enumerate(st["lens"].tolist()):
        t = torch.arange(max(0, n - st["window"]) if st["window"] else 0, n, device=DEV)
        if not n:
            continue
        page = st["table"][b].long()[t // ps]
        for g in range(hkv):
            k, v = (st[c + "pool"][g].view(torch.uint8 if st["cache"] != "f16" else torch.float16)[page * ps + t % ps].view(DTYPES[st["cache"]]).double() for c in "kv")
            if st["cache"] != "f16":
                k, v = k * st["kscale"][g].double()[page, None], v * st["vscale"][g].double()[page, None]
            heads = slice(g * (h // hkv), (g + 1) * (h // hkv))
            cost = None if slopes is None else slopes[g][:, None, None] * (n - 1 - t)[None, None]
            out[b, heads] = _attend(st["q"][b, heads].double()[:, None], k, v, st["softcap"], cost, None)[:, 0]
    return out


def _exact_pages(st):
    """The books kept by hand: a list of pages for each sequence."""
    ps, width = st["page"], st["table"].shape[1]
    table, lens, refs = (st[x].tolist() for x in ("table", "lens", "refs"))
    rows, n_pages, moves = [t[:-(-n // ps)] for t, n in zip(table, lens)], len(refs), []
    new_rows, new_lens, new_refs = [list(r) for r in rows], list(lens), list(refs)
    if st["kind"] == "fork":
        for b, p in enumerate(st["parents"].tolist()):
            new_rows[b], new_lens[b] = (list(rows[p]), lens[p]) if p >= 0 else ([], 0)
            for page in rows[b]:
                new_refs[page] -= 1
            for page in new_rows[b]:
                new_refs[page] += 1
    elif st["kind"] == "extend":
        add, free = st["add"].tolist(), [i for i, r in enumerate(refs) if r <= 0]
        writers, at, out_of_pages = {}, 0, False
        fits = [a > 0 and -(-(n + a) // ps) <= width for n, a in zip(lens, add)]
        for b, r in enumerate(rows):
            if fits[b] and lens[b] % ps:
                writers.setdefault(r[-1], []).append(b)
        for b, r in enumerate(rows):
            if add[b] < 0:
                new_lens[b] = max(0, lens[b] + add[b])
                new_rows[b] = r[:-(-new_lens[b] // ps)]
                for page in r[len(new_rows[b]):]:
                    new_refs[page] -= 1
            elif fits[b]:
                copy = bool(lens[b] % ps) and refs[r[-1]] > 1 and not (len(writers[r[-1]]) == refs[r[-1]] and writers[r[-1]][-1] == b)
                need = -(-(lens[b] + add[b]) // ps) - len(r) + copy
                out_of_pages |= need > 0 and at + need > len(free)
                if need > 0 and out_of_pages:
                    continue
                got, at = free[at:at + need], at + need
                if copy:
                    moves.append((r[-1], got[0], lens[b] % ps))
                    new_refs[r[-1]] -= 1
                    new_rows[b] = r[:-1] + got
                else:
                    new_rows[b] = r + got
                for page in got:
                    new_refs[page] = 1
                new_lens[b] += add[b]
    else:
        used = [i for i, r in enumerate(refs) if r > 0]
        where, holes = [-1] * n_pages, iter(i for i, r in enumerate(refs) if r <= 0)
        for i in used:
            where[i] = i if i < len(used) else next(holes)
            if where[i] != i:
                moves.append((i, where[i], ps))
        new_refs = [0] * n_pages
        for i in used:
            new_refs[where[i]] = refs[i]
        new_rows = [[where[page] for page in r] for r in rows]
    out = {"table": _int32([r + [0] * (width - len(r)) for r in new_rows]), "lens": _int32(new_lens), "refs": _int32(new_refs)}
    if st["kind"] == "compact":
        del out["lens"]
        out["where"] = _int32(where)
    if st["kind"] != "fork":
        for c in "kv":
            pool, scale = st[c + "pool"].clone(), st[c + "scale"]
            x = pool.view(torch.uint8) if scale is not None else pool
            scale = scale.clone() if scale is not None else None
            for a, b, n in moves:
                x[:, b * ps:b * ps + n] = x[:, a * ps:a * ps + n].clone()
                if scale is not None:
                    scale[:, b] = scale[:, a]
            out[c], out[c + "_scale"] = pool.double(), scale.double() if scale is not None else None
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_prompt(st) if case["kind"] == "prompt" else _exact_token(st) if case["kind"] == "token" else _exact_pages(st)


def work(case):
    kind = case["kind"]
    if kind == "prompt":
        n, h, hkv = case["tokens"], case["heads"], case["kv_heads"]
        docs = max(1, case["docs"])
        lengths = [n / docs] * docs if docs == 1 else [n * 2 * (i + 0.5) / docs ** 2 for i in range(docs)]      # unlike ones
        pairs, w = 0, case["window"] or n
        for m in lengths:
            pairs += m * (m + 1) / 2 if m <= w else w * (w + 1) / 2 + (m - w) * w
            pre = min(m, case["prefix"] / (2 if case["docs"] else 1))
            pairs += pre * (pre - 1) / 2 if pre > 1 else 0
        return {"bytes": 4 * D * n * (h + hkv), "flops": 4 * D * h * int(pairs)}
    ps = case["page"]
    if kind == "token":
        size, h, hkv = 2 if case["cache"] == "f16" else 1, case["heads"], case["kv_heads"]
        n = case["keys"] * (1 + 3 * (case["seqs"] - 1) / 4) / case["seqs"]                       # mean: uniform from half of it
        n = min(n, case["window"]) if case["window"] else n
        per_key = 2 * D * size + (8 / ps if size == 1 else 0)
        return {"bytes": case["seqs"] * (n * hkv * per_key + 4 * h * D + 4 * n / ps), "flops": 4 * D * h * case["seqs"] * n}
    # of four rows, two list the first one's pages, and one shares some of them: 1.1 times a longest row's pages in all
    b, mean, (pages, width) = case["seqs"], 0.75 * case["keys"], _sizes(case)
    books = b * 4 * (mean / ps + width + 3) + 8 * pages
    if kind == "fork":
        return {"bytes": books, "flops": 0}
    row = 2 * case["layers"] * case["kv_heads"] * D * (2 if case["cache"] == "f16" else 1)       # of keys and values of a token
    scale = 16 * case["layers"] * case["kv_heads"] if case["cache"] != "f16" else 0
    if kind == "extend":                                 # two of the three that share a page write to a copy of it, which is half full
        return {"bytes": books + 0.49 * b * (ps - 1) / ps * (2 * row * ps / 2 + scale), "flops": 0}
    used = 0.275 * b * case["keys"] / ps
    return {"bytes": books + 4 * pages + used * (1 - used / pages) * (2 * row * ps + scale), "flops": 0}
