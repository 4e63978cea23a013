"""The books of a paged cache kept by hand: a list of pages for each sequence, changed one sequence at a time."""


def pages(n, ps):
    return -(-n // ps)


def rows_of(table, lens, ps):
    return [r[:pages(n, ps)] for r, n in zip(table, lens)]


def fork(table, lens, refs, parents, ps):
    rows, refs = rows_of(table, lens, ps), list(refs)
    new = [list(rows[p]) if 0 <= p < len(rows) else [] for p in parents]
    for old, now in zip(rows, new):
        for page in old:
            refs[page] -= 1
        for page in now:
            refs[page] += 1
    return new, [lens[p] if 0 <= p < len(rows) else 0 for p in parents], refs


def extend(table, lens, refs, add, ps, width):
    """... and (page, its copy, rows of it) for each copy"""
    rows, before, refs, moves = rows_of(table, lens, ps), list(refs), list(refs), []
    free = [i for i, r in enumerate(before) if r <= 0]
    fits = [a > 0 and pages(n + a, ps) <= width and n + a < 1 << 31 for n, a in zip(lens, add)]
    writers = {}
    for b, r in enumerate(rows):
        if fits[b] and lens[b] % ps:
            writers.setdefault(r[-1], []).append(b)
    out, new_lens, at, short = [], [], 0, False
    for b, r in enumerate(rows):
        n, a = lens[b], add[b]
        if a <= 0:
            n = max(0, n + a)
            for page in r[pages(n, ps):]:
                refs[page] -= 1
            r = r[:pages(n, ps)]
        elif fits[b]:
            copy = n % ps != 0 and before[r[-1]] > 1 and not (len(writers[r[-1]]) == before[r[-1]] and writers[r[-1]][-1] == b)
            need = pages(n + a, ps) - len(r) + copy
            short = short or (need > 0 and at + need > len(free))
            if need == 0 or not short:
                got, at = free[at:at + need], at + need
                if copy:
                    moves.append((r[-1], got[0], n % ps))
                    refs[r[-1]] -= 1
                    r = r[:-1]
                for page in got:
                    refs[page] = 1
                r, n = r + got, n + a
        out.append(r)
        new_lens.append(n)
    return out, new_lens, refs, moves


def compact(table, lens, refs, ps):
    """... with where each page goes, and (page, where, rows of it) for each that moves"""
    used = [i for i, r in enumerate(refs) if r > 0]
    where, holes = [-1] * len(refs), iter(i for i, r in enumerate(refs) if r <= 0)
    for page in used:
        where[page] = page if page < len(used) else next(holes)
    new = [0] * len(refs)
    for page in used:
        new[where[page]] = refs[page]
    return [[where[page] for page in r] for r in rows_of(table, lens, ps)], new, where, [(i, where[i], ps) for i in used if where[i] != i]
