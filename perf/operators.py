"""Operators around a paged cache of keys and values, each one pass through its public entry point, and the same in
elementary torch operations.

  append   `page_append`: new tokens' keys are rotated to their positions and written, with their values, to the pages of
           their sequences, in fp16 or in 8 bits with a scale for each page and head; their queries are rotated beside.
           One token for each sequence (a decode step) or a ragged run of tokens for each (prompts, or chunks of them).
  q8       `page_flash_attn_q8`: one query for each sequence over pages held in 8 bits.
  window   `page_flash_attn` with a window: one query for each sequence over fp16 pages, of which it sees the last `window`
           keys and the first `sinks`.
  prompt   `causal_attn` with a window: the queries of a prompt, or of a later chunk of one, over its keys.

Heads, head size and page sizes are those of the 7B and 70B architectures that the package is written for and of its
tests; lengths go from a token to where windows and 8-bit caches are used for.
"""
from __future__ import annotations

import math

import torch

own = False

DEV, D, N_POS = "cuda", 128, 1 << 17
QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"f16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one sequence decodes its next token: latency and host time
        {"name": "append_1_f16", "kind": "append", "cache": "f16", "seqs": 1, "tokens": 1, "ragged": False, "heads": 32, "kv_heads": 32, "page": 16, "past": 512},
        # a decode step of many sequences with grouped heads, a page of each partly filled
        {"name": "append_100_e4m3", "kind": "append", "cache": "e4m3", "seqs": 100, "tokens": 100, "ragged": False, "heads": 32, "kv_heads": 8, "page": 16, "past": 512},
        # the prompts of five requests, some behind a part that is there already
        {"name": "append_prompts_f16", "kind": "append", "cache": "f16", "seqs": 5, "tokens": 4001, "ragged": True, "heads": 32, "kv_heads": 32, "page": 16, "past": 300},
        # a large batch of prompts of the 70B geometry into long pages
        {"name": "append_prompts_int8", "kind": "append", "cache": "int8", "seqs": 9, "tokens": 8191, "ragged": True, "heads": 64, "kv_heads": 8, "page": 64, "past": 100},
        # a short answer of one sequence
        {"name": "q8_1", "kind": "q8", "cache": "int8", "seqs": 1, "keys": 512, "heads": 32, "kv_heads": 32, "page": 16, "window": 0, "sinks": 0},
        # a full batch, lengths anywhere up to the longest
        {"name": "q8_64_e4m3", "kind": "q8", "cache": "e4m3", "seqs": 64, "keys": 2048, "heads": 32, "kv_heads": 32, "page": 16, "window": 0, "sinks": 0},
        # few very long sequences, eight query heads on each kv head
        {"name": "q8_long_int8", "kind": "q8", "cache": "int8", "seqs": 8, "keys": 65536, "heads": 64, "kv_heads": 8, "page": 64, "window": 0, "sinks": 0},
        # a narrow batch with a short window
        {"name": "window_10", "kind": "window", "cache": "f16", "seqs": 10, "keys": 2000, "heads": 32, "kv_heads": 32, "page": 16, "window": 256, "sinks": 4},
        # a full batch of long sequences, of which a window of 4096 is read
        {"name": "window_100", "kind": "window", "cache": "f16", "seqs": 100, "keys": 10000, "heads": 32, "kv_heads": 8, "page": 16, "window": 4096, "sinks": 4},
        # a short question, no multiple of anything
        {"name": "prompt_77", "kind": "prompt", "tokens": 77, "offset": 0, "heads": 32, "kv_heads": 32, "window": 50, "sinks": 4},
        # a later chunk of a long prompt
        {"name": "prompt_chunk", "kind": "prompt", "tokens": 2000, "offset": 6191, "heads": 32, "kv_heads": 32, "window": 1024, "sinks": 4},
        # a long prompt of the 70B geometry in one pass
        {"name": "prompt_16384", "kind": "prompt", "tokens": 16384, "offset": 0, "heads": 64, "kv_heads": 8, "window": 4096, "sinks": 4},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "q8", "window", "prompt"])
    heads, kv = rng.choice([(32, 32), (32, 8), (64, 8), (8, 1), (24, 6)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv}
    if kind == "prompt":
        case |= {"tokens": _log(rng, 1, 6000), "offset": rng.choice([0, _log(rng, 1, 8000)]), "sinks": rng.randint(0, 130)}
        return case | {"window": _log(rng, 1, 8192)}
    case["page"] = rng.choice([1, 16, 16, 20, 32, 64])
    if kind == "append":
        ragged, seqs = rng.random() < 0.5, _log(rng, 1, 100)
        tokens = max(seqs, _log(rng, 1, 8000)) if ragged else seqs
        return case | {"cache": rng.choice(list(DTYPES)), "seqs": seqs, "tokens": tokens, "ragged": ragged, "past": rng.randint(1, 512)}
    keys = _log(rng, 1, 32768)
    case |= {"seqs": min(_log(rng, 1, 128), max(1, 8 * 32768 * 8 // (keys * kv))), "keys": keys, "window": _log(rng, 1, 8192), "sinks": rng.randint(0, 64)}
    if kind == "window":
        return case | {"cache": "f16"}
    case["cache"] = rng.choice(["int8", "e4m3"])
    return case if rng.random() < 0.3 else case | {"window": 0, "sinks": 0}


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)


def _pool(gen, case, pages):
    """Pool and scales (None in fp16) of `pages` pages with keys or values of usual size, channels of unlike size among them."""
    x = _normal(gen, case["kv_heads"], pages * case["page"], D) * (0.5 + torch.rand((case["kv_heads"], 1, D), generator=gen, device=DEV)).half()
    if case["cache"] == "f16":
        return x, None
    x = x.view(case["kv_heads"], pages, case["page"], D)
    scale = x.abs().amax((2, 3)).float() / QMAX[case["cache"]]
    y = x.float() / scale[..., None, None]
    codes = y.round().to(torch.int8) if case["cache"] == "int8" else y.to(torch.float8_e4m3fn)
    return codes.view(case["kv_heads"], -1, D), scale


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _pages(gen, need, pages):
    """A table of page ids in any order out of `pages`, as many for each sequence as it needs (zeros behind them)."""
    need = torch.tensor(need)
    at = torch.arange(int(need.max()))[None] < need[:, None]
    table = torch.zeros(at.shape, dtype=torch.int32, device=DEV)
    table[at.to(DEV)] = torch.randperm(pages, generator=gen, device=DEV)[:int(need.sum())].to(torch.int32)
    return table


def prepare(case, seed):
    gen, host = torch.Generator(device=DEV).manual_seed(int(seed)), torch.Generator().manual_seed(int(seed))
    ints = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=host).tolist()
    h, hkv = case["heads"], case["kv_heads"]
    st = dict(case)
    if case["kind"] == "prompt":
        s, n = case["tokens"], case["tokens"] + case["offset"]
        return st | {"q": _normal(gen, s, h, D), "k": _normal(gen, n, hkv, D), "v": _normal(gen, n, hkv, D)}
    b, ps = case["seqs"], case["page"]
    if case["kind"] == "append":
        t = case["tokens"]
        cuts = sorted(torch.randperm(t - 1, generator=host)[:b - 1].add(1).tolist()) if case["ragged"] else list(range(1, b))
        offsets = [0] + cuts + [t]
        pos = ints(0, case["past"], b)
        if case["ragged"]:                      # about half of the prompts are whole ones
            pos = [0 if i else p for i, p in zip(ints(0, 1, b), pos)]
        pages = b * (case["past"] // ps + 2) + t // ps        # what any such batch finds room in
        table = _pages(gen, [(p + offsets[i + 1] - offsets[i] - 1) // ps + 1 for i, p in enumerate(pos)], pages)
        qkv = _normal(gen, t, (h + 2 * hkv), D)  # one projection's output: its queries, keys and values are views
        angle = torch.outer(torch.arange(N_POS, device=DEV).double(), 1e6 ** (-torch.arange(64, device=DEV).double() / 64))
        st |= {"q": qkv[:, :h], "k": qkv[:, h:h + hkv], "v": qkv[:, h + hkv:], "cos": angle.cos().half(), "sin": angle.sin().half(),
               "pos": _int32(pos), "offsets": _int32(offsets) if case["ragged"] else None}
    else:
        lens = [case["keys"]] + ints(case["keys"] // 2, case["keys"], b - 1)
        pages = b * -(-case["keys"] // ps)
        table = _pages(gen, [-(-n // ps) for n in lens], pages)
        st |= {"q": _normal(gen, b, h, D), "lens": _int32(lens), "longest": case["keys"]}
    st["table"] = table
    (st["kpool"], st["kscale"]), (st["vpool"], st["vscale"]) = _pool(gen, case, pages), _pool(gen, case, pages)
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _rotated(x, cos, sin):
    a, b = x[..., :64].float(), x[..., 64:].float()
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _append_8(st, pool, scale, x, slots):
    """Writes x [tokens, kv heads, D] to slots, pages' scales growing with what comes (in place)."""
    ps, top = st["page"], QMAX[st["cache"]]
    page, row = slots // ps, slots % ps
    first = torch.full_like(scale[0], ps).scatter_reduce(0, page, row.float(), "amin")           # of a page's new rows
    most = torch.zeros_like(scale).scatter_reduce(1, page[None].expand(scale.shape[0], -1), x.abs().amax(-1).t(), "amax")
    old = torch.where(first == 0, torch.zeros_like(scale), scale)
    new = torch.where(first < ps, torch.maximum(old, most * (1.0 / top)), scale)
    inv = torch.where(new > 0, 1.0 / new, torch.zeros_like(new))
    coded = lambda y: y.round().clamp(-top, top).to(pool.dtype) if pool.dtype == torch.int8 else y.clamp(-top, top).to(pool.dtype)
    pages = pool.view(scale.shape[0], -1, ps, D)
    there = (torch.arange(ps, device=DEV)[None] < first[:, None]) & (first < ps)[:, None] & ((new > old)[..., None])
    pages.copy_(torch.where(there[..., None], coded(pages.float() * (old * inv)[..., None, None]).float(), pages.float()).to(pool.dtype))
    pool.view(torch.uint8)[:, slots] = coded(x.transpose(0, 1) * inv[:, page][..., None]).view(torch.uint8)
    scale.copy_(new)


def _append_plain(st):
    n, ps = st["k"].shape[0], st["page"]
    at = torch.arange(n, device=DEV)
    seq = at if st["offsets"] is None else torch.searchsorted(st["offsets"][1:].contiguous(), at.int(), right=True)
    pos = st["pos"][seq].long() + (0 if st["offsets"] is None else at - st["offsets"][seq])
    slots = st["table"][seq, pos // ps].long() * ps + pos % ps
    cos, sin = st["cos"][pos], st["sin"][pos]
    k, v = _rotated(st["k"], cos, sin), st["v"].float()
    if st["kscale"] is None:
        st["kpool"][:, slots], st["vpool"][:, slots] = k.half().transpose(0, 1), st["v"].transpose(0, 1)
    else:
        _append_8(st, st["kpool"], st["kscale"], k, slots)
        _append_8(st, st["vpool"], st["vscale"], v, slots)
    return _rotated(st["q"], cos, sin).half()


def _visible(st):
    """Positions [sequences, most] of the keys that each sequence's query sees, and which of them are there."""
    n, w, sinks = st["lens"][:, None].long(), st["window"] or st["longest"], st["sinks"]
    lo = (n - w).clamp(min=0)
    first = lo.clamp(max=sinks)
    i = torch.arange(min(st["longest"], w + sinks), device=DEV)[None]
    return torch.where(i < first, i, i - first + lo), i < first + n - lo


def _decode_plain(st):
    ps, (b, h, _) = st["page"], st["q"].shape
    t, there = _visible(st)
    t = torch.where(there, t, 0)
    slots = st["table"].gather(1, t // ps).long() * ps + t % ps
    k, v = (x[:, slots].float() if s is None else x.view(torch.uint8)[:, slots].view(x.dtype).float() * s[:, slots // ps][..., None]
            for x, s in ((st["kpool"], st["kscale"]), (st["vpool"], st["vscale"])))             # [kv heads, sequences, keys, D]
    q = st["q"].float().view(b, k.shape[0], -1, D).transpose(0, 1)
    score = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(~there[:, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))                          # a sequence without keys: zeros
    return (e @ v / e.sum(-1, keepdim=True).clamp(min=1e-30)).transpose(0, 1).reshape(b, h, D).half()


def _prompt_plain(st, block=512):
    (s, h, _), off, w, sinks = st["q"].shape, st["offset"], st["window"], st["sinks"]
    hkv, out = st["k"].shape[1], torch.empty_like(st["q"])
    for a in range(0, s, block):
        e = min(s, a + block)
        lo = max(0, off + a - w + 1)
        j = torch.cat((torch.arange(min(sinks, lo), device=DEV), torch.arange(lo, off + e, device=DEV)))
        k, v = (x[j].float().permute(1, 2, 0) for x in (st["k"], st["v"]))                       # [kv heads, D, keys]
        q = st["q"][a:e].float().view(e - a, hkv, -1, D).permute(1, 2, 0, 3)                     # [kv heads, heads of one, queries, D]
        i = torch.arange(off + a, off + e, device=DEV)[:, None]
        seen = (j <= i) & ((i - j < w) | (j < sinks))
        score = (q @ k[:, None] / math.sqrt(D)).masked_fill(~seen, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        out[a:e] = (p @ v.transpose(1, 2)[:, None] / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).reshape(e - a, h, D).half()
    return out


def _cache_out(st):
    """The cache as it is held; 8-bit integers as the values that they stand for."""
    if st["cache"] != "int8":
        return {"k": st["kpool"], "v": st["vpool"], "k_scale": st["kscale"], "v_scale": st["vscale"]}
    out = {"k_scale": st["kscale"], "v_scale": st["vscale"]}
    for name in "kv":
        codes = st[name + "pool"].view(st["kv_heads"], -1, st["page"], D)
        out[name] = torch.mul(codes, st[name + "scale"][..., None, None], out=torch.empty(codes.shape, dtype=torch.float16, device=DEV))
    return out


def run(st):
    kind = st["kind"]
    if own:
        from spec_mcts_b200 import kernels as K
    if kind == "append":
        if own:
            q = K.page_append(st["table"], st["k"], st["v"], st["kpool"], st["vpool"], st["pos"], page_size=st["page"], offsets=st["offsets"],
                              k_scale=st["kscale"], v_scale=st["vscale"], q=st["q"], cos=st["cos"], sin=st["sin"])
        else:
            q = _append_plain(st)
        return {"q": q, **_cache_out(st)}
    if kind == "q8":
        if own:
            return K.page_flash_attn_q8(st["table"], st["q"], st["kpool"], st["vpool"], st["kscale"], st["vscale"], page_size=st["page"],
                                        seq_lens=st["lens"], window=st["window"] or None, sinks=st["sinks"])
        return _decode_plain(st)
    if kind == "window":
        if own:
            b, h, _ = st["q"].shape
            return K.page_flash_attn(st["table"], st["q"], st["kpool"], st["vpool"], st["kpool"].shape[1], b, st["longest"], h, D, page_size=st["page"],
                                     seq_lens=st["lens"], window=st["window"], sinks=st["sinks"])
        return _decode_plain(st)
    if own:
        return K.causal_attn(st["q"], st["k"], st["v"], window=st["window"], sinks=st["sinks"], offset=st["offset"])
    return _prompt_plain(st)


# ---- in 64 bits, sequence by sequence ------------------------------------------------------------------------------
def _attend(q, k, v, seen=None):
    """softmax(q k^T / sqrt(D)) v of [kv heads, rows, D] operands."""
    score = torch.bmm(q, k.transpose(1, 2)).div_(math.sqrt(D))
    if seen is not None:
        score = score.masked_fill_(~seen, -math.inf)
    return torch.bmm(torch.softmax(score, -1), v)


def _exact_append(st):
    ps, t, hkv = st["page"], st["k"].shape[0], st["kv_heads"]
    offsets = list(range(t + 1)) if st["offsets"] is None else st["offsets"].tolist()
    q, k, out = st["q"].double(), st["k"].double(), {}
    pools = {"k": st["kpool"].double(), "v": st["vpool"].double()}
    scales = {n: None if st[n + "scale"] is None else st[n + "scale"].double() for n in "kv"}
    at = torch.cat([torch.arange(b - a) + p for a, b, p in zip(offsets, offsets[1:], st["pos"].tolist())]).to(DEV)
    turn = torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
    rotate = lambda x: torch.view_as_real(torch.complex(x[..., :64], x[..., 64:]) * turn).movedim(-1, -2).flatten(-2)
    new = {"k": rotate(k), "v": st["v"].double()}
    table = st["table"].tolist()
    for i, (a, b) in enumerate(zip(offsets, offsets[1:])):
        p = int(st["pos"][i])
        while a < b:                                                       # a page of the sequence at a time
            row, page = p % ps, table[i][p // ps]
            n = min(ps - row, b - a)
            for name in "kv":
                x, rows = new[name][a:a + n].transpose(0, 1), pools[name][:, page * ps:(page + 1) * ps]
                if scales[name] is not None:
                    old = scales[name][:, page] if row else torch.zeros(hkv, dtype=torch.float64, device=DEV)
                    s = torch.maximum(old, x.abs().amax((1, 2)) / QMAX[st["cache"]])
                    held = (lambda y: y.round()) if st["cache"] == "int8" else (lambda y: y.to(torch.float8_e4m3fn).double())
                    rows[:, :row] = torch.where((s > old)[:, None, None], held(rows[:, :row] * (old / s)[:, None, None]), rows[:, :row])
                    x = held(x / s[:, None, None])
                    scales[name][:, page] = s
                rows[:, row:row + n] = x
            a, p = a + n, p + n
    for name in "kv":
        out[name] = pools[name]
        if st["cache"] == "int8":
            out[name] = pools[name].view(hkv, -1, ps, D) * scales[name][..., None, None]
    return {"q": rotate(q), **out, "k_scale": scales["k"], "v_scale": scales["v"]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(st)
    hkv = case["kv_heads"]
    if case["kind"] == "prompt":
        outs, (s, h, _), off, step = [], st["q"].shape, case["offset"], 1024
        for g in range(hkv):
            k, v, parts = st["k"][:, g].double()[None], st["v"][:, g].double()[None], []
            q = st["q"][:, g * (h // hkv):(g + 1) * (h // hkv)].double().transpose(0, 1)
            for a in range(0, s, step):
                i = torch.arange(a, min(s, a + step), device=DEV) + off
                lo, hi = max(0, int(i[0]) - case["window"] + 1), int(i[-1]) + 1
                lo = 0 if lo <= case["sinks"] else lo
                use = torch.arange(lo, hi, device=DEV)
                if lo:
                    use = torch.cat((torch.arange(case["sinks"], device=DEV), use))
                far = i[:, None] - use[None]
                seen = (far >= 0) & ((far < case["window"]) | (use < case["sinks"])[None])
                n = h // hkv
                parts.append(_attend(q[:, a:a + step], k[:, use].expand(n, -1, -1), v[:, use].expand(n, -1, -1), seen))
            outs.append(torch.cat(parts, 1).transpose(0, 1))
        return torch.cat(outs, 1)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    for i, n in enumerate(st["lens"].tolist()):
        t = torch.arange(n, device=DEV)
        if case["window"]:
            t = t[(n - 1 - t < case["window"]) | (t < case["sinks"])]
        page = st["table"][i].long()[t // case["page"]]
        slot = page * case["page"] + t % case["page"]
        k, v = (st[c + "pool"].view(torch.uint8 if case["cache"] != "f16" else torch.float16)[:, slot].view(DTYPES[case["cache"]]).double() for c in "kv")
        if case["cache"] != "f16":
            k, v = k * st["kscale"].double()[:, page, None], v * st["vscale"].double()[:, page, None]
        out[i] = _attend(st["q"][i].double().view(hkv, -1, D), k, v).reshape(-1, D)
    return out


def work(case):
    h, hkv = case["heads"], case["kv_heads"]
    if case["kind"] == "prompt":
        s, off, w, sinks = case["tokens"], case["offset"], case["window"], case["sinks"]
        pairs = 0
        for i in range(off, off + s):
            lo = max(0, i + 1 - w)
            pairs += i + 1 - lo + min(sinks, lo)
        first = max(0, off + 1 - w)                                       # keys that some query sees
        keys = off + s - first + min(sinks, first)
        return {"bytes": 4 * D * (s * h + keys * hkv), "flops": 4 * D * h * pairs}
    size = 2 if case["cache"] == "f16" else 1
    if case["kind"] == "append":
        t = case["tokens"]
        return {"bytes": t * (4 * h * D + 2 * hkv * D * (2 + size) + 256) + 8 * case["seqs"], "flops": 6 * t * (h + hkv) * 64}
    n = case["keys"] * (1 + 3 * (case["seqs"] - 1) / 4) / case["seqs"] if case["seqs"] > 1 else case["keys"]     # mean: uniform from half of it
    n = min(n, case["window"] + case["sinks"]) if case["window"] else n
    per_key = 2 * D * size + (8 / case["page"] if size == 1 else 0)
    return {"bytes": case["seqs"] * (n * hkv * per_key + 4 * h * D + 4 * n / case["page"]), "flops": 4 * D * h * case["seqs"] * n}
