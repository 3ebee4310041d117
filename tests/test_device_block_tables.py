"""DeviceBlockTables where requests find no room: the free list used up, a row
full, a step of more tokens than its buffers.  What a request is counted to have
is what the cache holds, in the steps after as well: on a model of the two kernels
(CPU) and on the kernels (GPU)."""
import math
import random

import numpy as np
import pytest
import torch

from _rows import assert_rows, attend64, tables64
from _util import pkg

BF16 = torch.bfloat16


def _model_tables(query, context, held, free, count, table, bs, max_tokens=None, out=None):
    """torch_ops.request_tables on CPU tensors, by the token-by-token reference."""
    t, n, left, start, lens, pos, slot = tables64(
        query.tolist(), context.tolist(), held.tolist(), free.tolist(), int(count),
        table.numpy(), bs, out.max_tokens)
    for dst, src in ((table, t), (out.num_pages, n), (out.free_count, [left]),
                     (out.query_start_loc, start), (out.seq_lens, lens), (out.positions, pos),
                     (out.slot_mapping, slot)):
        dst.copy_(torch.from_numpy(np.array(src)))
    return out


def _model_release(keep, held, free, count, table, bs):
    """torch_ops.release_pages on CPU tensors."""
    for r, k in enumerate(keep.tolist()):
        kept = min(-(-max(k, 0) // bs), int(held[r]))
        for b in range(kept, int(held[r])):
            free[int(count)] = table[r, b]
            count += 1
            table[r, b] = -1
        held[r] = kept


class _Buffers:
    """torch_ops.RequestTables without its checks that the buffers are on a GPU."""
    def __init__(self, reqs, max_tokens):
        i32 = dict(dtype=torch.int32)
        self.query_start_loc = torch.zeros(reqs + 1, **i32)
        self.seq_lens = torch.zeros(reqs, **i32)
        self.positions, self.slot_mapping = (torch.zeros(max_tokens, dtype=torch.int64)
                                             for _ in range(2))
        self.max_tokens = max_tokens

    def replace(self, num_pages, free_count):
        self.num_pages, self.free_count = num_pages, free_count
        return self


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def make(request, monkeypatch):
    """Makes DeviceBlockTables on the model or on the kernels."""
    mod = pkg("integration.block_table")
    if request.param == "cpu":
        ops = mod.torch_ops
        monkeypatch.setattr(ops, "request_tables", _model_tables)
        monkeypatch.setattr(ops, "release_pages", _model_release)
        monkeypatch.setattr(ops, "request_tables_out",
                            lambda n, max_tokens: _Buffers(n.numel(), max_tokens))
    return lambda *sizes: mod.DeviceBlockTables(*sizes, request.param)


class _Run:
    """DeviceBlockTables and what is in each slot: (request, position) of its writer."""
    def __init__(self, T, num_blocks, bs):
        self.T, self.bs = T, bs
        self.cache = [None] * (num_blocks * bs)

    def _i32(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.T.lens.device)

    def step(self, query):
        T = self.T
        context = T.lens.tolist()
        t = T.step(self._i32(query))
        rows = min(sum(query), t.positions.numel())
        owner = [r for r, n in enumerate(query) for _ in range(n)][:rows]
        pos, slot = t.positions.tolist(), t.slot_mapping.tolist()
        wrote = [0] * len(query)
        for j, r in enumerate(owner):
            if slot[j] >= 0:
                self.cache[slot[j]] = (r, pos[j])
                wrote[r] += 1
        # a request has what it had and the tokens that got a slot; the lengths of the
        # step count the rows that its buffers have room for
        assert T.lens.tolist() == [c + w for c, w in zip(context, wrote)], (query, context)
        assert t.seq_lens.tolist() == [c + owner.count(r) for r, c in enumerate(context)]
        self.check()
        return t

    def keep(self, lens):
        before = self.T.lens.tolist()
        self.T.keep(self._i32(lens))
        assert self.T.lens.tolist() == [min(a, max(b, 0)) for a, b in zip(before, lens)]
        self.check()

    def check(self):
        T, bs = self.T, self.bs
        table, pages = T.block_table.tolist(), T.num_pages.tolist()
        for r, L in enumerate(T.lens.tolist()):
            assert L <= pages[r] * bs
            for p in range(L):
                slot = table[r][p // bs] * bs + p % bs
                assert slot >= 0 and self.cache[slot] == (r, p), (r, p, self.cache[slot])
        held = [p for row, n in zip(table, pages) for p in row[:n]]
        free = T.free_pages.tolist()[:int(T.free_count)]
        assert sorted(held + free) == list(range(len(self.cache) // bs))


def test_a_token_without_a_page_is_not_counted(make):
    """A request that found the list empty does not get another's page for the lost
    token's place later: the token is not counted, and can be given again."""
    run = _Run(make(2, 32, 2, 4, 64), 2, 32)
    run.step([32, 32])
    t = run.step([1, 0])
    assert t.slot_mapping.tolist()[0] == -1 and run.T.lens.tolist() == [32, 32]
    run.keep([33, 0])
    t = run.step([1, 0])
    assert t.positions.tolist()[0] == 32 and t.slot_mapping.tolist()[0] >= 0
    assert run.T.lens.tolist() == [33, 0]


def test_some_tokens_of_a_prompt_without_a_page(make):
    run = _Run(make(3, 16, 2, 8, 100), 3, 16)
    run.step([20, 60])  # two pages, then one of the four
    assert run.T.lens.tolist() == [20, 16]
    run.keep([0, 16])
    run.step([0, 30])
    assert run.T.lens.tolist() == [0, 46]


def test_a_full_row(make):
    run = _Run(make(20, 16, 2, 3, 200), 20, 16)
    run.step([60, 40])
    run.step([5, 20])
    assert run.T.lens.tolist() == [48, 48]
    run.step([1, 1])
    run.keep([40, 0])
    run.step([8, 9])
    assert run.T.lens.tolist() == [48, 9]


def test_more_tokens_than_the_buffers_have_room_for(make):
    run = _Run(make(40, 16, 3, 10, 50), 40, 16)
    run.step([20, 40, 30])
    assert run.T.lens.tolist() == [20, 30, 0]
    run.step([0, 10, 30])
    assert run.T.lens.tolist() == [20, 40, 30]
    run.step([50, 1, 0])
    assert run.T.lens.tolist() == [70, 40, 30]


@pytest.mark.parametrize("seed", range(4))
def test_random_steps_short_of_room(make, seed):
    """Few pages, short rows, small buffers: every token that is counted is in the
    cache, as its own request wrote it, after every step."""
    r = random.Random(seed)
    S, bs, width, blocks, room = 5, 8, 5, 13, 40
    run = _Run(make(blocks, bs, S, width, room), blocks, bs)
    for _ in range(40):
        run.step([r.choice([0, 1, 1, 1, 3, 20, 45]) for _ in range(S)])
        if r.random() < 0.5:
            run.keep([r.choice([0, x, x, x + 4, max(0, x - 3), -1]) for x in run.T.lens.tolist()])


def test_sizes_that_int32_lengths_cannot_hold_are_refused(make):
    for sizes in ((4, 4096, 1, 1 << 19, 1), (4, 16, 1, 4, 2 ** 31 - 1), (0, 16, 1, 4, 8)):
        with pytest.raises(ValueError):
            make(*sizes)


@pytest.mark.gpu
def test_attention_after_the_list_ran_out():
    """Two requests' attention over a run in which the list is used up and a step
    is cut by its buffers: rows that see a token without a page are NaN in that
    step, all others are as float64 attention over the tokens that were kept."""
    ops, mod = pkg("native.torch_ops"), pkg("integration.block_table")
    bs, n_q, n_kv, hd, blocks, room = 32, 4, 1, 128, 4, 70
    g = torch.Generator().manual_seed(3)
    T = mod.DeviceBlockTables(blocks, bs, 2, 6, room, "cuda")
    kc, vc = (torch.full((blocks, bs, n_kv, hd), math.nan, dtype=BF16, device="cuda")
              for _ in range(2))
    kept = [[torch.zeros((0, n_kv, hd), dtype=BF16)] * 2 for _ in range(2)]

    def rand(*shape):
        return torch.randn(shape, generator=g).to(BF16)

    def step(n, lost=(0, 0)):
        t = T.step(torch.tensor(n, dtype=torch.int32, device="cuda"))
        rows = [max(0, min(n[0], room)), max(0, min(n[1], room - n[0]))]
        total = sum(rows)
        k, v, q = rand(total, n_kv, hd), rand(total, n_kv, hd), rand(total, n_q, hd)
        ops.reshape_and_cache(k.cuda(), v.cuda(), kc, vc, t.slot_mapping[:total])
        got = ops.prompt_attention(q.cuda(), kc, vc, T.block_table, t.query_start_loc, t.seq_lens,
                                   0.1).cpu()
        at = 0
        for r, m in enumerate(rows):
            have = m - lost[r]
            kept[r] = [torch.cat((a, b[at:at + have])) for a, b in zip(kept[r], (k, v))]
            L = kept[r][0].shape[0]
            if have:
                seen = torch.arange(L)[None] <= torch.arange(L - have, L)[:, None]
                ref, mag = attend64(q[at:at + have].double(), kept[r][0].double(),
                                    kept[r][1].double(), 0.1, seen)
                assert_rows(got[at:at + have], ref, mag, f"request {r} of {n}")
            assert torch.isnan(got[at + have:at + m]).all()
            at += m
        assert T.lens.tolist() == [x[0].shape[0] for x in kept]

    step([40, 25])               # two pages and one
    step([20, 10])               # the last page is request 1's
    step([5, 4], lost=(1, 0))
    T.keep(torch.tensor([64, 0], dtype=torch.int32, device="cuda"))
    kept[1] = [x[:0] for x in kept[1]]
    step([3, 2])
    step([1, 100], lost=(0, 39))  # 69 of its 100 rows, 30 in the one page it has


@pytest.mark.gpu
def test_captured_steps_short_of_room():
    """A captured step and keep, replayed on other lengths: the same tables, lengths and
    slots as another object's eager steps, where room runs out too."""
    mod = pkg("integration.block_table")
    S, r = 5, random.Random(9)
    a, b = (mod.DeviceBlockTables(13, 8, S, 5, 40, "cuda") for _ in range(2))
    query, keep = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(2))
    outs = []

    def run():
        outs.append(a.step(query))
        a.keep(keep)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(12):
        query.copy_(torch.tensor([r.choice([0, 1, 1, 9, 30]) for _ in range(S)]))
        keep.copy_(torch.tensor([r.choice([0, 7, 100, 100, 100]) for _ in range(S)]))
        graph.replay()
        want = b.step(query)
        b.keep(keep)
        torch.cuda.synchronize()
        for name in ("query_start_loc", "seq_lens", "positions", "slot_mapping"):
            assert torch.equal(getattr(outs[-1], name), getattr(want, name)), (i, name)
        for name in ("lens", "num_pages", "block_table", "free_count"):
            assert torch.equal(getattr(a, name), getattr(b, name)), (i, name)
