"""Pages that sequences share, one entry at a time (CPU): tables as lists of pages (None: absent), counts,
and pools as numpy arrays with the page first and the tokens on an axis of their own."""
import numpy as np

VALID = 1 << 31


def words(table, width):
    """A table as the int32 array that the calls take."""
    a = np.zeros((len(table), width), np.int64)
    for b, row in enumerate(table):
        for j, p in enumerate(row):
            if p is not None:
                a[b, j] = p | VALID
    return a.astype(np.uint32).view(np.int32)


def rows(array):
    """The reverse of words()."""
    return [[int(w) & (VALID - 1) if w < 0 else None for w in row] for row in array]


def counts(table, pages):
    c = [0] * pages
    for row in table:
        for p in row:
            if p is not None:
                c[p] += 1
    return c


def fork(table, refs, parents, width):
    out = [list(table[p]) if p >= 0 else [None] * width for p in parents]
    for t, by in ((out, 1), (table, -1)):
        for row in t:
            for p in row:
                if p is not None:
                    refs[p] += by
    return out


def reserve(table, refs, before, after, page, pools):
    """pools: (array, axis of the tokens, tokens that share an element).  Returns what was missing."""
    was = [list(r) for r in table], list(refs)
    free = [p for p, c in enumerate(refs) if c == 0]
    missing, moves = 0, []
    for b, (lo, hi) in enumerate(zip(before, after)):
        if hi <= lo:
            continue
        for j in range(lo // page, -(-hi // page)):
            had = table[b][j]
            if had is not None and refs[had] == 1:
                continue
            if not free:
                missing += 1
                if had is not None:
                    refs[had] -= 1
                continue
            new = free.pop(0)
            refs[new], table[b][j] = 1, new
            if had is not None:
                refs[had] -= 1
                if lo > j * page:
                    moves.append((had, new, lo - j * page))
    if missing:
        table[:], refs[:] = was
        return missing
    for a, axis, unit in pools:
        old = a.copy()
        for src, dst, n in moves:
            at = (slice(None),) * (axis - 1) + (slice(0, -(-n // unit)),)
            a[dst][at] = old[src][at]
    return 0


def release(table, refs, keep, page):
    for row, n in zip(table, keep):
        for j in range(-(-n // page), len(row)):
            if row[j] is not None:
                refs[row[j]] -= 1
                row[j] = None


def compact(table, refs, pools):
    n = sum(c > 0 for c in refs)
    src = [p for p in range(n, len(refs)) if refs[p]]
    dst = [p for p in range(n) if not refs[p]]
    to = dict(zip(src, dst))
    for row in table:
        row[:] = [to.get(p, p) for p in row]
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
        for pool, _, _ in pools:
            pool[b] = pool[a]
    return n
