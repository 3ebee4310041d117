"""What fork_pages and compact_pages do, row by row on the host."""
from __future__ import annotations


def fork(parents, lens, num_pages, free, table, num_blocks, bs):
    """-> (table, num_pages, lens, free list, copies), lists."""
    rows, width = len(table), len(table[0])
    pages = [min(max(n, 0), width) for n in num_pages]
    lens = [min(max(x, 0), n * bs) for x, n in zip(lens, pages)]
    kept = [-(-x // bs) for x in lens]
    inside = lambda p: 0 <= p < num_blocks  # noqa: E731
    before = {p for r in range(rows) for p in table[r][:pages[r]] if inside(p)}
    alive = {r for r in parents if 0 <= r < rows}
    live: dict[int, int] = {}
    for r in alive:
        for p in table[r][:kept[r]]:
            live[p] = live.get(p, 0) + 1
    free = list(free)
    out, out_pages, out_lens, copies, had = [], [], [], [], set()
    for r in parents:
        row, length, pair = [], 0, (-1, -1)
        if 0 <= r < rows:
            row, length = list(table[r][:kept[r]]), lens[r]
            if length % bs and inside(row[-1]) and (r in had or live[row[-1]] > 1):
                if free:
                    pair = (row[-1], free.pop())
                    row[-1] = pair[1]
                else:
                    row.pop()
                    length = len(row) * bs
                    # (the table's entry is -1 all the same)
            had.add(r)
        copies.append(list(pair))
        out_pages.append(len(row))
        out_lens.append(length)
        out.append(row + [-1] * (width - len(row)))
    after = {p for r, n in zip(out, out_pages) for p in r[:n]}
    return out, out_pages, out_lens, free + sorted(before - after), copies


def compact(num_pages, table, num_blocks):
    """-> (table, free list, moves), lists."""
    width = len(table[0])
    pages = [min(max(n, 0), width) for n in num_pages]
    used = sorted({p for r, n in zip(table, pages) for p in r[:n] if 0 <= p < num_blocks})
    holes = sorted(set(range(len(used))) - set(used))
    moves = [[p, holes[i]] for i, p in enumerate(q for q in used if q >= len(used))]
    to = {p: p for p in used} | {a: b for a, b in moves}
    out = [[to.get(p, -1) for p in r[:n]] + [-1] * (width - n) for r, n in zip(table, pages)]
    return out, list(range(num_blocks - 1, len(used) - 1, -1)), moves
