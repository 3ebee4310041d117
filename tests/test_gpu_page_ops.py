"""Pages that rows of the block tables share: fork_pages, compact_pages and copy_pages
against the same on the host."""
import random

import pytest
import torch

from _pages import compact, fork
from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ops():
    return pkg("native.torch_ops")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _state(rng, groups, beams, hi, bs, spare, width_more=2, shared=True):
    """Tables of `groups` searches whose beams share their first pages; tails are a row's own."""
    lens, table, used = [], [], 0
    for _ in range(groups):
        n = rng.randint(0, hi)
        held = -(-n // bs)
        common = rng.randint(0, max(held - 1, 0)) if shared else 0
        front = list(range(used, used + common))
        used += common
        for _ in range(beams):
            mine = list(range(used, used + held - common))
            used += held - common
            lens.append(n)
            table.append(front + mine)
    blocks = used + spare
    perm = list(range(blocks))
    rng.shuffle(perm)
    width = max(len(r) for r in table) + width_more
    pages = [len(r) for r in table]
    table = [[perm[p] for p in r] + [rng.choice([-1, 0, blocks + 9])] * (width - len(r))
             for r in table]
    return lens, pages, table, perm[used:], blocks


def _check(got, ref, count):
    table, pages, lens, free, copies = ref
    assert got.num_pages.tolist() == pages
    assert got.lens.tolist() == lens
    assert got.copies.tolist() == copies
    assert got.block_table.tolist() == table
    assert got.free_count.item() == min(len(free), count)
    assert got.free_pages.tolist() == (free + [-1] * count)[:count]


def _fork(parents, lens, pages, table, free, blocks, bs, count=None, out=None):
    count = count or blocks
    fp = _i32((free + [blocks - 1] * count)[:count])  # (entries past the count are not looked at)
    return _ops().fork_pages(_i32(parents), _i32(lens), _i32(pages), fp, _i32([len(free)]),
                             _i32(table), blocks, bs, out=out)


@pytest.mark.parametrize("groups,beams,hi,bs,spare", [
    (1, 1, 40, 16, 3), (1, 4, 100, 32, 8), (3, 5, 200, 16, 20), (64, 8, 900, 128, 600),
    (20, 2, 17, 1, 9), (5, 7, 2000, 4, 3), (300, 8, 64, 32, 2500), (1, 1100, 60, 16, 1200)])
@pytest.mark.parametrize("seed", range(3))
def test_fork_matches(groups, beams, hi, bs, spare, seed):
    rng = random.Random(seed * 1000 + groups)
    lens, pages, table, free, blocks = _state(rng, groups, beams, hi, bs, spare)
    rows = len(table)
    parents = [g * beams + rng.randrange(beams) for g in range(groups) for _ in range(beams)]
    if seed == 1:  # rows that end, and rows of another search's
        parents = [rng.choice([p, p, -1, rng.randrange(rows), rows + 3]) for p in parents]
    print(groups, beams, hi, bs, spare, seed, rows, blocks, flush=True)
    _check(_fork(parents, lens, pages, table, free, blocks, bs),
           fork(parents, lens, pages, free, table, blocks, bs), blocks)


def test_fork_over_several_steps():
    """A search of many steps: forks, growth by request_tables, and at the end every page
    but the last rows' is free, once."""
    ops, rng = _ops(), random.Random(5)
    beams, bs, blocks, width = 6, 4, 80, 9
    rows = 2 * beams
    table, lens, pages = torch.full((rows, width), -1, dtype=torch.int32, device="cuda"), \
        _i32([0] * rows), _i32([0] * rows)
    free, count = _i32(list(range(blocks))), _i32([blocks])
    # a prompt of 9 tokens in row 0, of 4 in row 6
    query = [9 if r == 0 else 4 if r == beams else 0 for r in range(rows)]
    parents = [0 if r < beams else beams for r in range(rows)]
    for step in range(12):
        t = ops.request_tables(_i32(query), lens, pages, free, count, table, bs, max_tokens=64)
        pages, count = t.num_pages, t.free_count
        before = [x.tolist() for x in (t.seq_lens, pages, table, free, count)]
        f = ops.fork_pages(_i32(parents), t.seq_lens, pages, free, count, table, blocks, bs)
        _check(f, fork(parents, before[0], before[1], before[3][:before[4][0]], before[2], blocks,
                       bs), blocks)
        table, lens, pages = f.block_table, f.lens, f.num_pages
        free, count = f.free_pages, f.free_count
        listed = {p for r, n in zip(table.tolist(), pages.tolist()) for p in r[:n]}
        left = free.tolist()[:count.item()]
        assert len(left) == len(set(left)) and not listed & set(left)
        assert sorted(listed | set(left)) == list(range(blocks)), f"step {step}"
        query = [1] * rows
        parents = [r // beams * beams + rng.randrange(beams) for r in range(rows)]


def test_fork_without_room():
    """Copies past the end of the free list: those rows are cut to their whole pages."""
    lens, pages = [70, 70, 20, 40], [5, 5, 2, 3]
    table = [[0, 1, 2, 3, 4], [0, 1, 2, 5, 6], [7, 8, -1, -1, -1], [9, 10, 11, -1, -1]]
    for room in range(4):
        free = [20, 21, 22][:room]
        args = ([0, 0, 2, 2], lens, pages, table, free, 30, 16)
        _check(_fork(*args), fork([0, 0, 2, 2], lens, pages, free, table, 30, 16), 30)


def test_fork_with_shared_tails_and_cut_rows():
    """Rows cut (lens below what they hold) into a page that another row lists: none of the
    two writes into the other's."""
    lens, pages = [20, 40, 18, 0], [3, 3, 3, 1]
    table = [[0, 1, 2], [0, 1, 3], [0, 1, 4], [5, -1, -1]]
    for parents in ([0, 1, 2, 3], [0, 0, 2, 2], [2, 2, 2, -1], [1, 1, 0, 0], [-1, -1, -1, -1],
                    [0, 2, 0, 2]):
        for free in ([9, 10, 11, 12], [9], []):
            _check(_fork(parents, lens, pages, table, free, 16, 16),
                   fork(parents, lens, pages, free, table, 16, 16), 16)


def test_fork_in_place_free_list_and_short_list():
    """The free list updated in place; a list too short for all pages drops the last ones."""
    rng = random.Random(8)
    lens, pages, table, free, blocks = _state(rng, 10, 4, 100, 16, 30)
    parents = [4 * (r // 4) + rng.randrange(4) for r in range(40)]
    ref = fork(parents, lens, pages, free, table, blocks, 16)
    ops = _ops()
    fp, fc, tab = _i32(free + [-1] * (blocks - len(free))), _i32([len(free)]), _i32(table)
    new = ops.fork_pages_out(tab, fp)
    out = ops.ForkedPages(new.block_table, new.num_pages, new.lens, fp, fc, new.copies)
    got = ops.fork_pages(_i32(parents), _i32(lens), _i32(pages), fp, fc, tab, blocks, 16, out=out)
    _check(got, ref, blocks)
    short = len(free) + 5
    _check(_fork(parents, lens, pages, table, free, blocks, 16, count=short), ref, short)


def test_fork_of_a_large_pool():
    """More pages and rows than the small kernel's sets hold."""
    rng = random.Random(9)
    lens, pages, table, free, blocks = _state(rng, 600, 4, 90, 16, 200000)
    parents = [4 * (r // 4) + rng.randrange(4) for r in range(len(table))]
    assert blocks > 32768 and len(table) > 2048
    _check(_fork(parents, lens, pages, table, free, blocks, 16),
           fork(parents, lens, pages, free, table, blocks, 16), blocks)


def _check_compact(got, ref, blocks):
    table, free, moves = ref
    assert got.block_table.tolist() == table
    assert got.free_count.item() == len(free)
    assert got.free_pages.tolist() == free + [-1] * (blocks - len(free))
    assert got.moves.tolist() == moves + [[-1, -1]] * (blocks // 2 - len(moves))


@pytest.mark.parametrize("groups,beams,hi,bs,spare", [
    (1, 1, 10, 16, 2), (3, 5, 200, 16, 20), (64, 8, 900, 128, 600), (5, 7, 2000, 4, 0),
    (2, 1, 0, 16, 7), (30, 1, 500, 16, 100000), (300, 8, 64, 32, 31)])
def test_compact_matches(groups, beams, hi, bs, spare):
    rng = random.Random(groups)
    _, pages, table, _, blocks = _state(rng, groups, beams, hi, bs, spare)
    blocks = max(blocks, 2)
    print(groups, beams, hi, bs, spare, blocks, flush=True)
    ref = compact(pages, table, blocks)
    tab = _i32(table)
    _check_compact(_ops().compact_pages(_i32(pages), tab, blocks), ref, blocks)
    assert tab.tolist() == table
    # in place
    ops = _ops()
    out = ops.CompactedPages(tab, _i32([0] * blocks), _i32([0]), _i32([[0, 0]] * (blocks // 2)))
    _check_compact(ops.compact_pages(_i32(pages), tab, blocks, out=out), ref, blocks)


def test_compact_leaves_entries_without_a_page():
    table = [[5, -1, 40], [3, 99, 6]]
    _check_compact(_ops().compact_pages(_i32([3, 3]), _i32(table), 41),
                   compact([3, 3], table, 41), 41)


@pytest.mark.parametrize("shapes,dtype,page_dim,pairs", [
    ([(2, 9, 32, 2, 64)] * 3, BF16, 1, [(0, 1), (-1, -1), (4, 8), (5, -1), (3, 99), (2, 2)]),
    ([(7, 32, 1, 64)], BF16, 0, [(6, 0)]),
    ([(2, 40, 8, 128, 64), (2, 40, 8, 128, 4)], torch.uint8, 1, [(i, 39 - i) for i in range(20)]),
    ([(3, 2, 300, 16)], torch.uint8, 2, [(i, i + 150) for i in range(150)])])
def test_copy_pages(shapes, dtype, page_dim, pairs):
    print(shapes, page_dim, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    caches = [torch.randint(0, 200, s, generator=g, device="cuda").to(dtype) for s in shapes]
    want = [c.clone() for c in caches]
    blocks = shapes[0][page_dim]
    for w in want:
        v = w.movedim(page_dim, 0)
        for a, b in pairs:
            if 0 <= a < blocks and 0 <= b < blocks:
                v[b] = v[a].clone()
    ops = _ops()
    ops.copy_pages(ops.PageSet(caches, page_dim), _i32(pairs))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)
    ops.copy_pages(ops.PageSet(caches, page_dim), _i32(pairs)[:0])


def test_capture_and_other_stream():
    """fork, copy and compact in one graph whose inputs change between replays."""
    ops, rng = _ops(), random.Random(11)
    bs, blocks = 16, 400
    cases = []
    while len(cases) < 4:
        lens, pages, table, free, b = _state(rng, 8, 4, 150, bs, 50, width_more=0)
        if b <= blocks and len(table[0]) <= 10:
            table = [r + [-1] * (10 - len(r)) for r in table]
            free = free + list(range(b, blocks))
            parents = [4 * (r // 4) + rng.randrange(4) for r in range(32)]
            cases.append((parents, lens, pages, table, free))
    cache = torch.randint(0, 255, (2, blocks, 64), dtype=torch.uint8, device="cuda")
    pages_of = ops.PageSet([cache])
    ins = [_i32(x) for x in cases[0][:4]]
    fp, fc = _i32([-1] * blocks), _i32([0])
    out = ops.fork_pages_out(ins[3], fp)
    copied = torch.empty_like(cache)

    def call():
        ops.fork_pages(ins[0], ins[1], ins[2], fp, fc, ins[3], blocks, bs, out=out)
        ops.copy_pages(pages_of, out.copies)
        copied.copy_(cache)
        c = ops.compact_pages(out.num_pages, out.block_table, blocks)
        ops.copy_pages(pages_of, c.moves)
        return c

    def load(case):
        for t, v in zip(ins, case[:4]):
            t.copy_(_i32(v))
        fp.copy_(_i32(case[4] + [-1] * (blocks - len(case[4]))))
        fc.copy_(_i32([len(case[4])]))

    load(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = call()
    for case in cases + cases[:1]:
        load(case)
        cache.random_(0, 255)
        was = cache.clone()
        graph.replay()
        torch.cuda.synchronize()
        ref = fork(case[0], case[1], case[2], case[4], case[3], blocks, bs)
        _check(out, ref, blocks)
        for a, b in ref[4]:
            if b >= 0:
                was[:, b] = was[:, a]
        assert torch.equal(copied, was)
        new = compact(ref[1], ref[0], blocks)
        _check_compact(c, new, blocks)
        for a, b in new[2]:
            was[:, b] = was[:, a]
        assert torch.equal(cache, was)


def test_refusals():
    ops = _ops()
    t = _i32([[0, 1], [2, -1]])
    a = dict(parents=_i32([0, 1]), lens=_i32([3, 2]), num_pages=_i32([2, 1]),
             free_pages=_i32([3, 4, -1]), free_count=_i32([2]), block_table=t, num_blocks=5,
             block_size=2)
    ops.fork_pages(**a)
    out = ops.fork_pages_out(t, a["free_pages"])
    bad = [dict(parents=_i32([0])), dict(parents=a["parents"].long()), dict(lens=_i32([3])),
           dict(num_pages=a["num_pages"].cpu()), dict(free_count=_i32([2, 2])),
           dict(block_table=t[0]), dict(block_table=t.long()), dict(out=(1, 2)),
           dict(out=out, free_pages=_i32([1, 2]))]
    for i, change in enumerate(bad):
        with pytest.raises(ValueError):
            ops.fork_pages(**{**a, **change})
            print("not refused:", i)
    Err = pkg("native").SmxError
    new = lambda **k: ops.ForkedPages(**{**{n: getattr(out, n) for n in out.__slots__}, **k})  # noqa: E731
    for change in (dict(out=new(block_table=t)), dict(out=new(num_pages=a["num_pages"])),
                   dict(out=new(lens=a["lens"])), dict(out=new(lens=a["num_pages"])),
                   dict(block_size=3), dict(num_blocks=0), dict(num_blocks=1 << 19)):
        with pytest.raises(Err):
            ops.fork_pages(**{**a, **change})
    with pytest.raises(ValueError):
        ops.compact_pages(_i32([2]), t, 5)
    with pytest.raises(ValueError):
        ops.compact_pages(_i32([2, 1]), t, 1)
    cache = torch.zeros((2, 5, 16), dtype=torch.uint8, device="cuda")
    for tensors, dim in (([], 1), ([cache.cpu()], 1), ([cache, cache[:, :4].contiguous()], 1),
                         ([cache[..., :8].contiguous()], 1), ([cache[:, :, ::2]], 1), ([cache], 3),
                         ([cache], -1)):
        with pytest.raises(ValueError):
            ops.PageSet(tensors, dim)
    s = ops.PageSet([cache])
    for pairs in (_i32([0, 1]), _i32([[0, 1, 2]]), _i32([[0, 1]]).long(), _i32([[0, 1]]).cpu()):
        with pytest.raises(ValueError):
            ops.copy_pages(s, pairs)
    with pytest.raises(ValueError):
        ops.copy_pages([cache], _i32([[0, 1]]))


@pytest.mark.parametrize("rows", [3, 20, 90])
def test_any_tables(rows):
    """Pages listed in any way: twice in a row, as the full page of one and the last of another,
    none at all, entries outside the pool; lengths below and above what rows hold."""
    rng = random.Random(rows)
    for _ in range(25):
        bs, width = rng.choice([1, 4, 16]), rng.randint(1, 6)
        blocks = rng.randint(2, 3 * rows)
        table = [[rng.choice([rng.randrange(blocks), rng.randrange(blocks), -1, blocks])
                  for _ in range(width)] for _ in range(rows)]
        pages = [rng.randint(-1, width + 1) for _ in range(rows)]
        lens = [rng.randint(-2, (width + 1) * bs) for _ in range(rows)]
        listed = {p for r, n in zip(table, pages) for p in r[:max(n, 0)]}
        free = [p for p in range(blocks) if p not in listed]
        rng.shuffle(free)
        parents = [rng.randint(-1, rows) for _ in range(rows)]
        _check(_fork(parents, lens, pages, table, free, blocks, bs),
               fork(parents, lens, pages, free, table, blocks, bs), blocks)
        got = _ops().compact_pages(_i32(pages), _i32(table), blocks)
        out, left, moves = compact(pages, table, blocks)
        assert got.block_table.tolist() == out
        assert got.free_count.item() == len(left)
        assert got.free_pages.tolist() == left + [-1] * (blocks - len(left))
        assert got.moves.tolist() == (moves + [[-1, -1]] * blocks)[:blocks // 2]
