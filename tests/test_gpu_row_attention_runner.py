"""The row attentions and the request tables recorded by the step runner, with the
attentions reading the tables, offsets and lengths that the same recording writes:
every replay on other inputs and poisoned buffers, so that a packet that starts
before the one it depends on, or reads what an earlier replay left, shows."""
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("hd,bs", [(128, 64), (64, 32)])
def test_replays_on_other_inputs(hd, bs):
    ops, runner = pkg("native.torch_ops"), pkg("native.runner")
    S, n_q, n_kv, rows, width, pages = 3, 8, 2, 12, 3200 // bs, 10000 // bs
    g = torch.Generator(device="cuda").manual_seed(3)
    i32 = dict(dtype=torch.int32, device="cuda")
    kc, vc = (torch.randn((pages, bs, n_kv, hd), generator=g, device="cuda").to(BF16)
              for _ in range(2))
    q = torch.empty((rows, n_q, hd), dtype=BF16, device="cuda")
    q2 = torch.empty((S, n_q, hd), dtype=BF16, device="cuda")
    query, context, held, count, plen = (torch.zeros(n, **i32) for n in (S, S, S, 1, 1))
    free = torch.empty(pages, **i32)
    inputs = (q, q2, query, context, free, count, plen)

    class Buffers:
        def __init__(self):
            self.table = torch.empty((S, width), **i32)
            self.tabs = ops.request_tables_out(held, rows)
            self.out, self.out2 = torch.empty_like(q), torch.empty_like(q2)
            self.ws = ops.prompt_attention_workspace(q, kc, self.table)
            self.ws2 = ops.shared_prefix_attention_workspace(q2, kc, self.table[0], self.table)

        def results(self):
            t = self.tabs
            return (self.table, t.query_start_loc, t.seq_lens, t.positions, t.slot_mapping,
                    t.num_pages, t.free_count, self.out, self.out2)

        def poison(self):
            self.table.fill_(-1)
            for x in self.results()[1:]:
                x.fill_(-3)
            for x in (self.ws, self.ws2):
                x.fill_(255)

        def run(self):
            t = self.tabs
            ops.request_tables(query, context, held, free, count, self.table, bs, out=t)
            ops.prompt_attention(q, kc, vc, self.table, t.query_start_loc, t.seq_lens, 0.1,
                                 workspace=self.ws, out=self.out)
            ops.shared_prefix_attention(q2, kc, vc, self.table[0], plen, self.table, t.seq_lens,
                                        0.1, workspace=self.ws2, out=self.out2)

    def set_inputs(n, c, prefix):
        q.normal_(generator=g)
        q2.normal_(generator=g)
        free.copy_(torch.randperm(pages, generator=g, device="cuda"))
        count.fill_(pages)
        plen.fill_(prefix)
        query.copy_(torch.tensor(n))
        context.copy_(torch.tensor(c))

    a = Buffers()
    assert a.ws is not None and a.ws2 is not None
    set_inputs([1, 1, 1], [5, 5, 5], 3)
    a.poison()
    a.run()
    torch.cuda.synchronize()
    steps = [([4, 3, 5], [3000, 10, 900], 700), ([1, 0, 11], [40, 0, 3], 41),
             ([2, 9, 0], [1500, 2900, 2000], 1502), ([4, 3, 5], [0, 0, 0], 0),
             ([5, 5, 2], [3100, 2500, 1], 3105), ([12, 0, 0], [800, 3000, 64], 64)]
    with runner.StepRunner() as r:
        r.record(a.run)
        for fences in ("agent", "acquire"):
            for step in steps:
                print(fences, step, flush=True)
                set_inputs(*step)
                a.poison()
                b = Buffers()
                b.poison()
                b.run()
                torch.cuda.synchronize()
                before = [x.clone() for x in inputs]
                torch.cuda.synchronize()
                r.run(1, fences=fences)
                torch.cuda.synchronize()
                for x, y in zip(a.results(), b.results()):
                    assert torch.equal(x, y), (fences, step)
                for x, y in zip(inputs, before):
                    assert torch.equal(x, y)
