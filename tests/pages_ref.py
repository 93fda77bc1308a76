"""Plain forms of the plans over a pool's pages, as loops over rows and pages."""


def forks(parents, lens, table, free, head, P, keep=None):
    """Lists in, a dict of lists out.  For steps that fit."""
    B, W = len(lens), len(table[0])
    n = [0 if p < 0 else lens[p] if keep is None else min(keep[i], lens[p]) for i, p in enumerate(parents)]
    whole, begun = set(), {}
    for i, p in enumerate(parents):
        whole |= {table[p][c] for c in range(n[i] // P)}
    for i, p in sorted(enumerate(parents), key=lambda x: (x[1] != x[0], x[0])):
        if n[i] % P and table[p][n[i] // P] not in whole:
            begun.setdefault(table[p][n[i] // P], i)
    out, copies = [], []
    for i, p in enumerate(parents):
        row = [table[p][c] for c in range(n[i] // P)]
        if n[i] % P:
            page = table[p][n[i] // P]
            if begun.get(page) != i:
                copies.append([page, free[head], n[i] % P, 0])
                page, head = free[head], head + 1
            row.append(page)
        out.append(row + [0] * (W - len(row)))
    held = {table[i][c] for i in range(B) for c in range(-(-lens[i] // P))}
    back = sorted(held - whole - set(begun))
    free = list(free)
    head -= len(back)
    free[head:head + len(back)] = back
    return dict(block_table=out, seq_lens=n, free_pages=free, free_head=[head], copies=copies + [[0] * 4] * (B - len(copies)))


def compaction(lens, table, P, N):
    slots = [0] * N
    for n, row in zip(lens, table):
        for c in range(-(-n // P)):
            slots[row[c]] = max(slots[row[c]], min(P, n - c * P))
    used = sum(s > 0 for s in slots)
    moving = [p for p in range(used, N) if slots[p]]
    holes = [p for p in range(used) if not slots[p]]
    to = dict(zip(moving, holes))
    W = len(table[0])
    out = [[to.get(p, p) for p in row[:-(-n // P)]] + [0] * (W - -(-n // P)) for n, row in zip(lens, table)]
    copies = [[p, to[p], slots[p], 0] for p in moving]
    return dict(block_table=out, free_pages=list(range(N)), free_head=[used], copies=copies + [[0] * 4] * (N // 2 - len(copies)))
