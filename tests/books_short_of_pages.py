"""Extension of the books of a paged cache as books_by_hand.extend, also where pages run out: who keeps a page that others were to copy counts as one that wants pages, so that it is
refused behind a sequence that is, which may still list that page."""
import books_by_hand as hand


def extend(table, lens, refs, add, ps, width):
    rows, new_refs, moves = hand.rows_of(table, lens, ps), list(refs), []
    free = [i for i, r in enumerate(refs) if r <= 0]
    grows = [a > 0 and hand.pages(n + a, ps) <= width and n + a < 1 << 31 for n, a in zip(lens, add)]
    tails = [r[-1] if g and n % ps and refs[r[-1]] > 1 else None for r, g, n in zip(rows, grows, lens)]         # shared, and to be written to
    new_rows, new_lens, at, refused = [], [], 0, False
    for b, (row, n, a, tail) in enumerate(zip(rows, lens, add, tails)):
        if a <= 0:
            n = max(0, n + a)
            given_back = row[hand.pages(n, ps):]
            row = row[:hand.pages(n, ps)]
            for page in given_back:
                new_refs[page] -= 1
        elif grows[b]:
            keeps = tail is not None and tails.count(tail) == refs[tail] and tail not in tails[b + 1:]
            copies = tail is not None and not keeps
            need = hand.pages(n + a, ps) - len(row) + copies
            refused |= at + need > len(free)
            if not refused or not (need or keeps):
                got, at = free[at:at + need], at + need
                for page in got:
                    new_refs[page] = 1
                if copies:
                    moves.append((tail, got[0], n % ps))
                    new_refs[tail] -= 1
                    row = row[:-1]
                row, n = row + got, n + a
        new_rows.append(row)
        new_lens.append(n)
    return new_rows, new_lens, new_refs, moves
