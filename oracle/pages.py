"""Oracle: a cache's pages by their reference counts, and rows and pages moved (CPU, plain loops, test infrastructure).
Tables, counts and lengths are lists that the calls change, as the operators change their tensors."""
from __future__ import annotations


def pages_for(positions: int, page_size: int) -> int:
    return -(-max(positions, 0) // page_size)


def _take(refs, asks):
    """The lowest free pages for `asks` pages a request, in order; None from the first that does not fit on."""
    free = [p for p, n in enumerate(refs) if n == 0]
    out, at, dry = [], 0, False
    for n in asks:
        if n == 0:
            out.append([])
        elif dry or at + n > len(free):
            dry = True
            out.append(None)
        else:
            out.append(free[at:at + n])
            at += n
    return out


def reserve(refs, table, length, target, page_size: int):
    """granted per request."""
    first = [pages_for(n, page_size) for n in length]
    asks = [max(pages_for(t, page_size) - f, 0) for t, f in zip(target, first)]
    fits = [f + n <= len(row) or n == 0 for f, n, row in zip(first, asks, table)]
    got = _take(refs, [n if ok else 0 for n, ok in zip(asks, fits)])
    for row, f, pages in zip(table, first, got):
        for j, p in enumerate(pages or []):
            row[f + j] = p
            refs[p] = 1
    return [int(ok and g is not None) for ok, g in zip(fits, got)]


def release(refs, table, length, keep, page_size: int) -> bool:
    """False where a page was given back that nobody held."""
    fine = True
    for b, row in enumerate(table):
        for j in range(pages_for(keep[b], page_size) if keep is not None else 0, min(pages_for(length[b], page_size), len(row))):
            p, row[j] = row[j], -1
            if 0 <= p < len(refs):
                fine &= refs[p] > 0
                refs[p] -= refs[p] > 0
    return fine


def fork(refs, table, length, parent, child, page_size: int):
    """(granted, pages to copy [(src, dst, slots)])."""
    rows, width = len(table), len(table[0]) if table else 0
    good = [0 <= p < rows and 0 <= c < rows and p != c and pages_for(length[p], page_size) <= width for p, c in zip(parent, child)]
    got = _take(refs, [int(ok and max(length[p], 0) % page_size > 0) if ok else 0 for ok, p in zip(good, parent)])
    granted, copies = [], []
    for ok, pages, p, c in zip(good, got, parent, child):
        granted.append(int(ok and pages is not None))
        if not granted[-1]:
            continue
        full = max(length[p], 0) // page_size
        for j in range(full):
            table[c][j] = table[p][j]
            if 0 <= table[p][j] < len(refs):
                refs[table[p][j]] += 1
        for page in pages:
            refs[page] = 1
            table[c][full] = page
            copies.append((table[p][full], page, length[p] % page_size))
        length[c] = max(length[p], 0)
    return granted, copies


def keep_path(pools, table, base, path, length, page_size: int) -> None:
    """pools: tensors [pages, heads, page_size, ...], changed in place."""
    pages = len(pools[0])

    def slot(b, pos):
        if pos < 0 or pos >= len(table[b]) * page_size or not 0 <= table[b][pos // page_size] < pages:
            return None
        return table[b][pos // page_size], pos % page_size

    for pool in pools:
        old = pool.clone()
        for b, row in enumerate(path):
            for j in range(min(max(length[b], 0), len(row))):
                src, dst = (slot(b, base[b] + row[j]) if row[j] >= 0 else None), slot(b, base[b] + j)
                if src is not None and dst is not None:
                    pool[dst[0], :, dst[1]] = old[src[0], :, src[1]]


def copy_pages(pools, src, dst, slots) -> None:
    for pool in pools:
        old, pages = pool.clone(), len(pool)
        for i, (a, b) in enumerate(zip(src, dst)):
            if 0 <= a < pages and 0 <= b < pages and a != b:
                n = pool.shape[2] if slots is None else min(max(slots[i], 0), pool.shape[2])
                pool[b, :, :n] = old[a, :, :n]
