"""Pages dealt and returned, one after the other, on the host."""


def assign(table, lengths, new, free, count, page, T):
    """Changes table and free (lists) in place; returns (cu, positions, slots, missing, count)."""
    n_pages, width = len(free), len(table[0]) if table else 0
    count = min(max(count, 0), n_pages)
    cu, positions, slots, missing = [0], [], [], 0
    for row, h, m in zip(table, lengths, new):
        m = min(m, T - cu[-1]) if h >= 0 and m > 0 else 0
        cu.append(cu[-1] + m)
        if m > 0:
            for i in range(h // page, min(width, (h + m - 1) // page + 1)):
                if not 0 <= row[i] < n_pages:
                    if count > 0:
                        count -= 1
                        row[i] = free[count]
                    else:
                        missing += 1
        for at in range(h, h + m):
            i = at // page
            positions.append(min(at, 2 ** 31 - 1))
            there = i < width and 0 <= row[i] < n_pages
            slots.append(row[i] * page + at % page if there else -1)
    positions += [-1] * (T - cu[-1])
    slots += [-1] * (T - cu[-1])
    return cu, positions, slots, missing, count


def release(table, lengths, free, count, page, window=None, sinks=0):
    """Changes table and free in place; returns count."""
    n_pages = len(free)
    count = min(max(count, 0), n_pages)
    back = []
    for row, keep in zip(table, lengths):
        for i, x in enumerate(row):
            a, b = i * page, (i + 1) * page
            gone = a >= keep or (window is not None and a >= sinks and b <= keep + 1 - window)
            if keep >= 0 and 0 <= x < n_pages and gone:
                back.append(x)
                row[i] = -1
    for k, x in enumerate(back):
        at = count + len(back) - 1 - k
        if at < n_pages:
            free[at] = x
    return min(count + len(back), n_pages)
