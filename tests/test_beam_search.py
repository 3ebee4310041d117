"""Beam search through a cache in 4 bits (integration.beam.BeamSearch): the operators
together, against the same attention over a cache of each row's own, written anew from its
tokens each step."""
import pytest
import torch

from _util import pkg

BF16 = torch.bfloat16
BS, N_Q, N_KV, HD, VOCAB = 32, 8, 2, 128, 1009


class Tables:
    """What BeamSearch's checks look at."""
    def __init__(self, rows, pages):
        self.lens = torch.zeros(rows, dtype=torch.int32)
        self.free_pages = torch.zeros(pages, dtype=torch.int32)


@pytest.mark.parametrize("rows,beams", [(6, 4), (4, 0), (65, 65)])
def test_rows_of_beams(rows, beams):
    with pytest.raises(ValueError, match="beams"):
        pkg("integration.beam").BeamSearch(Tables(rows, 4), None, beams)


def test_pages_must_be_a_page_set():
    with pytest.raises(ValueError, match="PageSet"):
        pkg("integration.beam").BeamSearch(Tables(4, 4), [torch.zeros(4)], 4)


def test_sequences_follow_the_parents():
    search = object.__new__(pkg("integration.beam").BeamSearch)
    search.beams, search.done = 2, torch.zeros(4, dtype=torch.bool)
    search._history = [(torch.tensor([0, 0, 2, -1]), torch.tensor([5, 6, 7, 0])),
                       (torch.tensor([1, 0, 2, 2]), torch.tensor([8, 9, 10, 11]))]
    assert search.sequences().tolist() == [[[6, 8], [5, 9]], [[7, 10], [7, 11]]]
    assert search.query_lens().tolist() == [1, 1, 1, 1]


class Model:
    """A layer: K, V and Q of a token by its id and place, read from tables, so that they do
    not depend on the rows of a call; logits by one product."""
    def __init__(self, device):
        g = torch.Generator(device=device).manual_seed(5)
        rand = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
        self.tab = [rand(VOCAB, n, HD).to(BF16) for n in (N_Q, N_KV, N_KV)]
        self.place = [rand(512, n, HD).to(BF16) for n in (N_Q, N_KV, N_KV)]
        self.head = (rand(VOCAB, N_Q * HD) / 8).to(BF16)

    def qkv(self, tokens, positions):
        return [(t[tokens] + p[positions]).flatten(1) for t, p in zip(self.tab, self.place)]

    def logits(self, out):
        return torch.nn.functional.linear(out, self.head)


def meta(step, table, seq_lens):
    mod = pkg("integration.attention")
    return mod.SplitKVDecodeMetadata(block_tables=table, seq_lens=seq_lens,
                                     slot_mapping=step[0], num_splits=1, query_start_loc=step[1])


@pytest.mark.gpu
@pytest.mark.parametrize("beams,prompts,eos,compact_every", [
    (1, [33], -1, 0), (4, [45, 64, 1], -1, 3), (8, [31, 70], 17, 5), (3, [95, 2], 17, 1)])
def test_run_together(beams, prompts, eos, compact_every):
    ops, att, tab = pkg("native.torch_ops"), pkg("integration.attention"), pkg("integration.block_table")
    beam = pkg("integration.beam")
    print(beams, prompts, eos, compact_every, flush=True)
    dev, steps = "cuda", 36
    rows, width = len(prompts) * beams, -(-(max(prompts) + steps) // BS)
    blocks = rows * width + 3
    model = Model(dev)
    impl = att.SplitKVDecodeBackend.get_impl_cls()(N_Q, HD, HD ** -0.5, N_KV)
    cache = att.SplitKVDecodeBackend.get_q4_kv_cache(blocks, BS, N_KV, HD, dev)
    tables = tab.DeviceBlockTables(blocks, BS, rows, width, sum(prompts), dev)
    search = beam.BeamSearch(tables, ops.PageSet(cache.planes()), beams, eos)
    g = torch.Generator().manual_seed(1)
    texts = [[]] * rows
    for s, n in enumerate(prompts):
        texts[s * beams] = torch.randint(0, VOCAB, (n,), generator=g).tolist()

    # the other cache: row r has the pages r * width, ..
    own_cache = ops.q4_kv_cache(rows * width, BS, N_KV, HD, dev)
    own_table = torch.arange(rows * width, dtype=torch.int32, device=dev).view(rows, width)

    def own(q, start, takes):
        """The attention of the rows' last tokens, `takes` of each, from the texts."""
        tokens = torch.tensor([t for x in texts for t in x], device=dev)
        place = torch.tensor([i for x in texts for i in range(len(x))], device=dev)
        slots = torch.tensor([r * width * BS + i for r, x in enumerate(texts)
                              for i in range(len(x))], device=dev)
        _, k, v = model.qkv(tokens, place)
        ops.reshape_and_cache_q4(k.view(-1, N_KV, HD), v.view(-1, N_KV, HD), own_cache, slots)
        lens = torch.tensor([len(x) if n else 0 for x, n in zip(texts, takes)],
                            dtype=torch.int32, device=dev)
        out = torch.zeros_like(q).view(-1, N_Q, HD)
        return ops.q4_attention(q.view(-1, N_Q, HD), own_cache, own_table, lens, HD ** -0.5,
                                query_start_loc=start, out=out).view(q.shape)

    takes = [len(x) for x in texts]
    feed = torch.tensor([t for x in texts for t in x], device=dev)
    for n in range(steps):
        step = tables.step(torch.tensor(takes, dtype=torch.int32, device=dev))
        count = sum(takes)
        q, k, v = model.qkv(feed[:count], step.positions[:count])
        m = meta((step.slot_mapping[:count], step.query_start_loc), tables.block_table,
                 torch.where(torch.tensor(takes, device=dev) > 0, step.seq_lens, 0))
        out = impl.forward(None, q, k, v, cache, m)
        want = own(q, step.query_start_loc, takes)
        assert torch.equal(out, want), f"step {n}"
        logits = torch.zeros((rows, VOCAB), dtype=BF16, device=dev)
        ends = step.query_start_loc[1:].long() - 1
        live = torch.tensor([r for r in range(rows) if takes[r]], device=dev)
        logits[live] = model.logits(out[ends[live]])
        before = search.done.tolist()
        tokens = search.step(logits)
        parents = search._history[-1][0].tolist()
        texts = [texts[p] + ([] if before[p] else [t]) if p >= 0 else []
                 for p, t in zip(parents, tokens.tolist())]
        if compact_every and n % compact_every == 0:
            ops.copy_pages(search.pages, tables.compact())
        takes = search.query_lens().tolist()
        if not sum(takes):
            break
        feed = tokens[torch.tensor(takes, device=dev) > 0]
        held = [len(x) - 1 if takes[r] else len(x) for r, x in enumerate(texts)]
        # (a beam that is done has its last token in its text alone)
        lens = tables.lens.tolist()
        assert all(a == b for a, b, k in zip(lens, held, takes) if k)
        # every page once: in rows that share it, or free
        pages = {p for r, c in zip(tables.block_table.tolist(), tables.num_pages.tolist())
                 for p in r[:c]}
        left = tables.free_pages[:int(tables.free_count)].tolist()
        assert not pages & set(left)
        assert sorted(pages | set(left)) == list(range(blocks))
        if compact_every == 1:
            assert sorted(pages) == list(range(len(pages)))
    got = search.sequences().view(rows, -1).tolist()
    for r in range(rows):
        if search.scores.view(-1)[r] > float("-inf"):
            made = texts[r][prompts[r // beams]:]
            assert got[r][:len(made)] == made and set(got[r][len(made):]) <= {0}
    scores = search.scores
    assert (scores[:, :-1] >= scores[:, 1:]).all()


@pytest.mark.gpu
def test_keep_is_refused_after_a_fork():
    tab = pkg("integration.block_table")
    t = tab.DeviceBlockTables(8, BS, 2, 4, 64, "cuda")
    t.step(torch.tensor([40, 0], dtype=torch.int32, device="cuda"))
    t.keep(torch.tensor([33, 0], dtype=torch.int32, device="cuda"))
    copies = t.fork(torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
    assert copies.tolist() == [[-1, -1], [1, 2]]
    assert t.lens.tolist() == [33, 33] and t.block_table.tolist() == [[0, 1, -1, -1], [0, 2, -1, -1]]
    with pytest.raises(RuntimeError, match="fork"):
        t.keep(torch.tensor([33, 0], dtype=torch.int32, device="cuda"))
    t.fork(torch.tensor([-1, 1], dtype=torch.int32, device="cuda"))
    assert t.lens.tolist() == [0, 33] and int(t.free_count) == 6


@pytest.mark.gpu
def test_a_cache_in_4_bits_has_no_plan():
    ops, att = pkg("native.torch_ops"), pkg("integration.attention")
    cache = ops.q4_kv_cache(2, BS, N_KV, HD, "cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    m = att.SplitKVDecodeMetadata(torch.zeros((1, 1), **i32), torch.ones(1, **i32),
                                  torch.zeros(1, dtype=torch.int64, device="cuda"), 1,
                                  prefix_table=torch.zeros(1, **i32))
    impl = att.SplitKVDecodeImpl(N_Q, HD, 1.0, N_KV)
    with pytest.raises(ValueError, match="4 bits"):
        impl.forward(None, torch.zeros((1, N_Q * HD), dtype=BF16, device="cuda"), None, None,
                     cache, m)


@pytest.mark.gpu
def test_a_captured_fork_and_compaction():
    """DeviceBlockTables.fork and compact captured before any other call of theirs, with the
    copies, and replayed; against the same calls one by one."""
    ops, tab = pkg("native.torch_ops"), pkg("integration.block_table")
    rows, blocks = 4, 24
    i32 = dict(dtype=torch.int32, device="cuda")

    def fresh():
        t = tab.DeviceBlockTables(blocks, BS, rows, 4, 200, "cuda")
        cache = ops.q4_kv_cache(blocks, BS, N_KV, HD, "cuda")
        cache.codes.copy_(torch.arange(cache.codes.numel(), device="cuda").view(cache.codes.shape))
        return t, cache, ops.PageSet(cache.planes())

    (a, ca, pa), (b, cb, pb) = fresh(), fresh()
    parents = torch.zeros(rows, **i32)
    ones = torch.ones(rows, **i32)

    def turn(t, pages):
        ops.copy_pages(pages, t.fork(parents))
        ops.copy_pages(pages, t.compact())

    for t in (a, b):
        t.step(torch.tensor([40, 64, 1, 0], **i32))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn(a, pa)
    for p in ([0, 0, 1, 2], [1, 1, 1, 2], [3, 2, -1, 0], [0, 0, 0, 0], [2, 1, 0, 3]):
        parents.copy_(torch.tensor(p))
        graph.replay()
        turn(b, pb)
        for t in (a, b):
            t.step(ones)
        torch.cuda.synchronize()
        for x, y in ((a.block_table, b.block_table), (a.num_pages, b.num_pages), (a.lens, b.lens),
                     (a.free_pages, b.free_pages), (a.free_count, b.free_count),
                     (ca.codes, cb.codes)):
            assert torch.equal(x, y), p
