"""Block tables, slots, positions and offsets from request lengths on the device
(torch_ops.request_tables) and the return of pages (release_pages): exact."""
import random

import numpy as np
import pytest
import torch

from _rows import tables64
from _util import pkg

pytestmark = pytest.mark.gpu


def _ops():
    return pkg("native.torch_ops")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _state(seed, context, width, bs, free):
    """A table that holds the context's pages, and a shuffled free list of `free`."""
    r = random.Random(seed)
    held = [min(-(-max(c, 0) // bs), width) for c in context]
    pages = list(range(sum(held) + free))
    r.shuffle(pages)
    table = np.full((len(context), width), -1, np.int32)
    for i, h in enumerate(held):
        for b in range(h):
            table[i, b] = pages.pop()
    return table, held, pages


def _check(query, context, width, bs, free, max_tokens, seed=0, capacity=None, in_place=False):
    table, held, left = _state(seed, context, width, bs, free)
    cap = capacity or max(len(left), 1)
    fp = _i32(left + [-9] * (cap - len(left)))
    t, n, c = _i32(table.tolist()), _i32(held), _i32([len(left)])
    ops = _ops()
    out = ops.request_tables_out(n, max_tokens)
    if in_place:
        out = out.replace(num_pages=n, free_count=c)
    got = ops.request_tables(_i32(query), _i32(context), n, fp, c, t, bs, out=out)
    want = tables64(query, context, held, left, len(left), table, bs, max_tokens)
    for name, a, b in zip(("table", "num_pages", "free_count", "query_start_loc", "seq_lens",
                           "positions", "slot_mapping"),
                          (t, got.num_pages, got.free_count, got.query_start_loc, got.seq_lens,
                           got.positions, got.slot_mapping), want):
        a = a.cpu().numpy().reshape(-1)
        b = np.array(b).reshape(-1)
        assert np.array_equal(a, b), (name, a, b)
    return t, got, fp


CASES = [
    # query, context, width, bs, free, max_tokens
    ([1], [0], 1, 1, 1, 1),
    ([1], [0], 4, 128, 3, 1),
    ([1] * 16, [(37 * i) % 400 for i in range(16)], 5, 128, 20, 16),
    ([0, 5, 0, 130, 1], [0, 127, 3, 0, 128], 4, 32, 30, 150),
    ([0, 0], [0, 0], 2, 32, 1, 4),
    ([-3, 4], [10, 0], 3, 16, 2, 9),
    ([500], [1], 9, 64, 9, 501),
    ([(11 * i) % 70 for i in range(300)], [(7 * i) % 90 for i in range(300)], 7, 32, 900, 11000),
    ([(11 * i) % 4 for i in range(2500)], [(7 * i) % 9 for i in range(2500)], 4, 4, 4000, 4000),
    ([3000, 5000], [100, 7], 100, 128, 70, 8100),
    ([4096], [0], 33, 128, 40, 4096),
    ([4097], [0], 33, 128, 40, 4097),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("in_place", [False, True])
def test_exact(case, in_place):
    print(f"tables case {str(case)[:150]}", flush=True)
    _check(*case, in_place=in_place)


@pytest.mark.parametrize("names", [("free_count",), ("num_pages",)])
def test_half_in_place(names):
    """One of the two updated in place, the other not, over many tokens."""
    query, context = [900, 0, 5000, 1], [3, 700, 64, 31]
    table, held, left = _state(4, context, 90, 64, 100)
    t, n, c, fp = _i32(table.tolist()), _i32(held), _i32([len(left)]), _i32(left)
    own = dict(free_count=c, num_pages=n)
    ops = _ops()
    out = ops.request_tables_out(n, 6000).replace(**{k: own[k] for k in names})
    got = ops.request_tables(_i32(query), _i32(context), n, fp, c, t, 64, out=out)
    want = tables64(query, context, held, left, len(left), table, 64, 6000)
    for a, b in zip((t, got.num_pages, got.free_count, got.query_start_loc, got.seq_lens,
                     got.positions, got.slot_mapping), want):
        assert np.array_equal(a.cpu().numpy().reshape(-1), np.array(b).reshape(-1)), names


def test_list_used_up_and_row_full():
    """Requests past the end of the free list get -1, and so do tokens past the
    table's row; pages there are not taken."""
    _check([40, 40, 40], [0, 0, 20], 4, 16, 4, 130)
    _check([300, 5], [0, 0], 2, 16, 10, 310)
    _check([300, 5], [0, 0], 2, 16, 0, 310, capacity=1)


def test_padding_shorter_than_the_tokens():
    """max_tokens below the tokens: what fits is written, the offsets are whole."""
    _check([10, 10], [0, 5], 2, 16, 9, 13)
    _check([5000, 10], [0, 5], 320, 16, 400, 4500)


def test_counts_and_pages_out_of_range_are_clamped():
    ops = _ops()
    t = torch.full((2, 3), 5, dtype=torch.int32, device="cuda")
    r = ops.request_tables(_i32([4, 4]), _i32([0, 0]), _i32([-4, 99]), _i32([7, 8]), _i32([50]),
                           t, 4, max_tokens=8)
    assert r.num_pages.tolist() == [1, 3] and r.free_count.tolist() == [1]
    assert t.tolist() == [[8, 5, 5], [5, 5, 5]]
    assert r.slot_mapping.tolist() == [32, 33, 34, 35, 20, 21, 22, 23]


def test_lengths_near_the_top_of_int32():
    ops = _ops()
    big = 2 ** 31 - 1
    t = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    r = ops.request_tables(_i32([big, big, 2]), _i32([big, 0, 5]), _i32([0, 0, 0]), _i32([1, 2]),
                           _i32([2]), t, 4096, max_tokens=3)
    assert r.query_start_loc.tolist() == [0, big, big, big]
    assert r.seq_lens.tolist() == [big, big, 7]
    assert r.positions.tolist() == [big, big + 1, big + 2]
    assert r.slot_mapping.tolist() == [-1, -1, -1]


def test_random_steps_with_releases():
    """A run of steps as a server makes them: tokens come, drafts are taken back,
    requests finish; no page is ever held twice, none is lost."""
    ops = _ops()
    r = random.Random(3)
    S, bs, width, total = 9, 16, 12, 100
    n, t = _i32([0] * S), torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    fp, c = _i32(list(range(total))), _i32([total])
    lens = [0] * S
    for step in range(25):
        query = [min(r.choice([0, 1, 1, 5, 40]), width * bs - x) for x in lens]
        out = ops.request_tables_out(n, 400).replace(num_pages=n, free_count=c)
        got = ops.request_tables(_i32(query), _i32(lens), n, fp, c, t, bs, out=out)
        lens = [a + b for a, b in zip(lens, query)]
        assert got.seq_lens.tolist() == lens
        if step % 3 == 2:
            lens = [r.choice([0, x, max(0, x - 3), x // 2]) for x in lens]
            ops.release_pages(_i32(lens), n, fp, c, t, bs)
        held = [p for row, k in zip(t.tolist(), n.tolist()) for p in row[:k]]
        free = fp.tolist()[:int(c)]
        if -1 not in held:
            assert sorted(held + free) == list(range(total))
        assert all(p == -1 for row, k in zip(t.tolist(), n.tolist()) for p in row[k:])
        assert n.tolist() == [-(-x // bs) for x in lens]


@pytest.mark.parametrize("S", [3, 300, 1500])
def test_release_order(S):
    """Pages come back in request and block order; entries become -1."""
    ops = _ops()
    width, bs = 4, 8
    table = [[100 * i + b for b in range(width)] for i in range(S)]
    held = [(i * 3) % (width + 1) for i in range(S)]
    keep = [(i * 5) % 37 for i in range(S)]
    t, n = _i32(table), _i32(held)
    fp, c = _i32([-7] * (S * width + 2)), _i32([2])
    ops.release_pages(_i32(keep), n, fp, c, t, bs)
    kept = [min(-(-k // bs), h) for k, h in zip(keep, held)]
    back = [table[i][b] for i in range(S) for b in range(kept[i], held[i])]
    assert n.tolist() == kept and int(c) == 2 + len(back)
    assert fp.tolist()[2:2 + len(back)] == back
    assert t.tolist() == [[table[i][b] if not kept[i] <= b < held[i] else -1
                           for b in range(width)] for i in range(S)]


def test_release_into_a_full_list_drops_the_rest():
    ops = _ops()
    t, n, fp, c = _i32([[1, 2], [3, 4]]), _i32([2, 2]), _i32([9, 9, 9]), _i32([1])
    ops.release_pages(_i32([0, -5]), n, fp, c, t, 8)
    assert fp.tolist() == [9, 1, 2] and c.tolist() == [3] and n.tolist() == [0, 0]


def test_captured_and_replayed():
    """A recorded step that keeps its pages in place, replayed on new lengths."""
    ops = _ops()
    S, bs, width = 20, 16, 30
    n, t = _i32([0] * S), torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    fp, c = _i32(list(range(500))), _i32([500])
    query, context = _i32([0] * S), _i32([0] * S)
    out = ops.request_tables_out(n, 6000).replace(num_pages=n, free_count=c)
    call = lambda: ops.request_tables(query, context, n, fp, c, t, bs, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    lens = [0] * S
    for i in range(4):
        q = [(7 * j + 31 * i) % 100 for j in range(S)]
        query.copy_(_i32(q))
        context.copy_(_i32(lens))
        held, left, tab = n.tolist(), fp.tolist()[:int(c)], t.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        want = tables64(q, lens, held, left, len(left), tab, bs, 6000)
        assert np.array_equal(t.cpu().numpy(), want[0]) and n.tolist() == want[1]
        assert int(c) == want[2] and out.slot_mapping.tolist() == want[6]
        lens = want[4]


def test_wrapper_refusals():
    ops = _ops()
    ok = dict(query_lens=_i32([1, 1]), context_lens=_i32([0, 0]), num_pages=_i32([0, 0]),
              free_pages=_i32([1, 2]), free_count=_i32([2]), block_table=_i32([[0], [0]]),
              block_size=16, max_tokens=2)
    ops.request_tables(**ok)
    for change in (dict(query_lens=_i32([1])), dict(context_lens=_i32([1, 2]).long()),
                   dict(free_count=_i32([1, 2])), dict(block_table=_i32([0, 0])),
                   dict(free_pages=_i32([])), dict(max_tokens=None), dict(max_tokens=0),
                   dict(num_pages=_i32([0, 0]).cpu())):
        with pytest.raises(ValueError):
            ops.request_tables(**{**ok, **change})
    with pytest.raises(pkg("native").SmxError):
        ops.request_tables(**{**ok, "block_size": 24})
    with pytest.raises(pkg("native").SmxError):  # lengths are not updated in place
        out = ops.request_tables_out(ok["num_pages"], 2).replace(seq_lens=ok["context_lens"])
        ops.request_tables(**{**ok, "max_tokens": None, "out": out})
