"""Page tables of a cache in pages, by walking the rows (lists of whole numbers; semantics: include/slotpage.h), and the pages' contents
as dense sequences."""
import torch


def up(n, page):
    return -(-n // page)


def extend(new, lens, table, free, page, N):
    """Changes lens, table (a list of rows) and free in place; (starts, ends, slots, pos)."""
    P, M = len(free) - 1, len(table[0])
    n = left = min(max(free[0], 0), P)
    starts, ends, slots, pos = [0], [], [-1] * N, [-1] * N
    at = asked = 0
    for r, want in enumerate(new):
        want = max(want, 0)
        first, have = at, lens[r]
        at += want
        starts.append(min(at, N))
        fits = want > 0 and at <= N and have >= 0 and have + want <= M * page
        need = up(have + want, page) - up(have, page) if fits else 0
        asked += need
        if not fits or (need and asked > n):
            ends.append(0)
            continue
        for i in range(need):
            table[r][up(have, page) + i] = free[left]
            left -= 1
        lens[r] = have + want
        ends.append(lens[r])
        for t in range(want):
            p = have + t
            pos[first + t] = p
            if 0 <= table[r][p // page] < P:
                slots[first + t] = table[r][p // page] * page + p % page
    free[0] = left
    return starts, ends, slots, pos


def trim(keep, lens, table, free, page):
    """Changes lens, table and free in place."""
    back = []
    for r, k in enumerate(keep):
        have = min(max(lens[r], 0), len(table[r]) * page)
        lens[r] = min(max(k, 0), have)
        for i in range(up(lens[r], page), up(have, page)):
            back.append(table[r][i])
            table[r][i] = -1
    n = min(max(free[0], 0), len(free) - 1)
    for x in reversed(back):
        n += 1
        if n < len(free):
            free[n] = x
    free[0] = min(n, len(free) - 1)


def dense(pages, ids, n):
    """The first n rows of a sequence in pages (P, H, page, D): (1, H, n, D); rows of pages outside of the pool: 0."""
    P, H, page, D = pages.shape
    out = torch.zeros(1, H, n, D, dtype=pages.dtype)
    for j in range(0, n, page):
        i = int(ids[j // page])
        if 0 <= i < P:
            m = min(page, n - j)
            out[0, :, j: j + m] = pages[i, :, :m]
    return out
