"""A cache in 4 bits, beam selection and the pages' operators recorded by the step runner,
each reading what the ones before it in the recording write: every replay on other inputs
and poisoned buffers, against the same calls made one after another."""
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("hd,bs,rows_each", [(128, 32, 1), (64, 64, 3), (128, 64, 90)])
def test_replays_on_other_inputs(hd, bs, rows_each):
    ops, runner = pkg("native.torch_ops"), pkg("native.runner")
    seqs, beams, n_q, n_kv, vocab, width = 2, 4, 8, 2, 20011, 2048 // bs
    rows = seqs * beams
    pages, tokens = rows * width + 40, rows * rows_each
    g = torch.Generator(device="cuda").manual_seed(3)
    i32 = dict(dtype=torch.int32, device="cuda")
    q, k, v = (torch.empty((tokens, n, hd), dtype=BF16, device="cuda") for n in (n_q, n_kv, n_kv))
    slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
    lens, held, count = torch.empty(rows, **i32), torch.empty(rows, **i32), torch.empty(1, **i32)
    table, free = torch.empty((rows, width), **i32), torch.empty(pages, **i32)
    start = torch.arange(0, tokens + 1, rows_each, **i32)
    scores = torch.empty(rows, dtype=torch.float32, device="cuda")
    done = torch.zeros(rows, dtype=torch.bool, device="cuda")
    logits = torch.empty((rows, vocab), dtype=BF16, device="cuda")
    codes = torch.empty((2, pages, n_kv, bs, hd // 2), dtype=torch.uint8, device="cuda")

    class Buffers:
        def __init__(self):
            self.cache = ops.q4_kv_cache(pages, bs, n_kv, hd, "cuda")
            self.pages = ops.PageSet(self.cache.planes())
            self.out = torch.empty_like(q)
            self.ws = ops.q4_attention_workspace(q, self.cache, table)
            self.best = ops.beam_select_out(seqs, beams, "cuda")
            self.ws2 = ops.beam_select_workspace(logits, beams, beams)
            self.fork = ops.fork_pages_out(table, free)
            self.packed = ops.CompactedPages(torch.empty_like(table), torch.empty_like(free),
                                             torch.empty(1, **i32), torch.empty((pages // 2, 2), **i32))

        def results(self):
            f, c, b = self.fork, self.packed, self.best
            return (self.cache.codes, self.cache.scales.view(torch.int16), self.out, b.parents,
                    b.tokens, b.scores, f.block_table, f.num_pages, f.lens, f.free_pages,
                    f.free_count, f.copies, c.block_table, c.free_pages, c.free_count, c.moves)

        def poison(self):
            self.cache.codes.copy_(codes)
            self.cache.scales.fill_(0.25)
            for x in self.results()[2:]:
                x.fill_(-3)
            for x in (self.ws, self.ws2):
                if x is not None:
                    x.fill_(255)

        def run(self):
            ops.reshape_and_cache_q4(k, v, self.cache, slots)
            ops.q4_attention(q, self.cache, table, lens, 0.1, query_start_loc=start,
                             workspace=self.ws, out=self.out)
            b = ops.beam_select(logits, scores, beams, beams, done=done, workspace=self.ws2,
                                out=self.best)
            f = ops.fork_pages(b.parents.view(-1), lens, held, free, count, table, pages, bs,
                               out=self.fork)
            ops.copy_pages(self.pages, f.copies)
            c = ops.compact_pages(f.num_pages, f.block_table, pages, out=self.packed)
            ops.copy_pages(self.pages, c.moves)

    def set_inputs(new_lens, ended):
        for x in (q, k, v, logits):
            x.normal_(generator=g)
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device="cuda"))
        scores.uniform_(-3, 0, generator=g)
        done.fill_(False)
        done[ended] = True
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table.fill_(-1)
        used = 0
        for r, n in enumerate(new_lens):
            m = -(-n // bs)
            table[r, :m] = order[used:used + m]
            for i in range(rows_each):
                at = n - rows_each + i
                slots[r * rows_each + i] = table[r, at // bs].long() * bs + at % bs
            used += m
            held[r] = m
            lens[r] = n
        free.fill_(-1)
        free[:pages - used] = order[used:]
        count.fill_(pages - used)

    steps = [([100 + 90 * r for r in range(rows)], []), ([bs * (3 + r) for r in range(rows)], [1, 6]),
             ([2048 - 7 * r for r in range(rows)], [0, 1, 2, 3]), ([97] * rows, [])]
    a = Buffers()
    set_inputs(*steps[0])
    a.poison()
    a.run()
    torch.cuda.synchronize()
    with runner.StepRunner() as r:
        r.record(a.run)
        for fences in ("agent", "acquire"):
            for step in steps:
                print(fences, step, flush=True)
                set_inputs(*step)
                b = Buffers()
                b.poison()
                b.run()
                a.poison()
                torch.cuda.synchronize()
                r.run(1, fences=fences)
                torch.cuda.synchronize()
                for i, (x, y) in enumerate(zip(a.results(), b.results())):
                    assert torch.equal(x, y), (fences, step, i)


def test_custom_ops():
    ops = pkg("native.torch_ops")
    pkg("integration.custom_ops").register()
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = ops.q4_kv_cache(4, 32, 2, 128, "cuda")
    k, v = (torch.randn((100, 2, 128), generator=g, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn((3, 8, 128), generator=g, device="cuda").to(BF16)
    slots = torch.arange(100, device="cuda")
    ops.reshape_and_cache_q4(k, v, cache, slots)
    table = torch.arange(4, dtype=torch.int32, device="cuda").repeat(3, 1)
    lens = torch.tensor([100, 1, 33], dtype=torch.int32, device="cuda")
    want = ops.q4_attention(q, cache, table, lens, 0.1)
    got = torch.ops.smx.q4_attention(q, cache.codes, cache.scales, table, lens, 0.1)
    assert torch.equal(got, want)
    start = torch.tensor([0, 1, 1, 3], dtype=torch.int32, device="cuda")
    got = torch.ops.smx.q4_attention(q, cache.codes, cache.scales, table, lens, 0.1, start)
    assert torch.equal(got, ops.q4_attention(q, cache, table, lens, 0.1, query_start_loc=start))
    x = torch.randn((6, 1000), generator=g, device="cuda").to(BF16)
    c = torch.zeros(6, device="cuda")
    want = ops.beam_select(x, c, 3, 5)
    got = torch.ops.smx.beam_select(x, c, 3, 5)
    for a, b in zip(got, (want.parents, want.tokens, want.scores)):
        assert torch.equal(a, b)
    fn = torch.compile(lambda a, b: torch.ops.smx.beam_select(a, b, 3, 5)[1] + 1, backend="eager",
                       fullgraph=True)
    assert torch.equal(fn(x, c), want.tokens + 1)
