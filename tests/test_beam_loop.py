"""Beam search's loop without the host: the tokens that a step's tables pack, and where the
rows' logits are among theirs."""
import pytest
import torch

from _util import pkg
from test_beam_search import BS, HD, N_KV, N_Q, Model, meta

BF16 = torch.bfloat16


@pytest.mark.parametrize("done,want", [
    ([0, 0, 0, 0], [5, 6, 7, 8]), ([1, 0, 0, 1], [6, 7, 9, 9]), ([0, 1, 1, 0], [5, 8, 9, 9]),
    ([1, 1, 1, 1], [9, 9, 9, 9])])
def test_packed_tokens(done, want):
    search = object.__new__(pkg("integration.beam").BeamSearch)
    search.pad_id, search.done = 9, torch.tensor(done, dtype=torch.bool)
    search._history = []
    with pytest.raises(RuntimeError, match="first step"):
        search.packed_tokens()
    search._history = [(None, torch.tensor([1, 2, 3, 4])), (None, torch.tensor([5, 6, 7, 8]))]
    got = search.packed_tokens()
    assert got.dtype == torch.int64 and got.tolist() == want

    class Tables:
        query_start_loc = torch.tensor([0, *(1 - search.done.long()).cumsum(0)], dtype=torch.int32)

    at = search.last_rows(Tables)
    assert at.dtype == torch.int64
    for r in range(4):
        assert done[r] or got[at[r]] == 5 + r
        assert 0 <= at[r] < 4


@pytest.mark.gpu
@pytest.mark.parametrize("beams,prompts,eos", [(4, [45, 64, 1], 17), (3, [95, 2], 100), (2, [7], -1)])
def test_a_loop_without_the_host(beams, prompts, eos):
    """Against the same search with the ended beams' tokens taken out on the host."""
    ops, att, tab = pkg("native.torch_ops"), pkg("integration.attention"), pkg("integration.block_table")
    dev, steps, rows = "cuda", 24, len(prompts) * beams
    width = -(-(max(prompts) + steps) // BS)
    print(beams, prompts, eos, flush=True)
    model = Model(dev)
    model.head[eos] *= 3  # (so that some beams end)
    head = model.head.double().t().contiguous()
    impl = att.SplitKVDecodeBackend.get_impl_cls()(N_Q, HD, HD ** -0.5, N_KV)
    g = torch.Generator().manual_seed(2)
    feed = torch.randint(0, 1009, (sum(prompts),), generator=g).to(dev)
    lens = torch.zeros(rows, dtype=torch.int32)
    lens[::beams] = torch.tensor(prompts, dtype=torch.int32)
    lens = lens.to(dev)

    def run(host):
        blocks = rows * width
        cache = att.SplitKVDecodeBackend.get_q4_kv_cache(blocks, BS, N_KV, HD, dev)
        tables = tab.DeviceBlockTables(blocks, BS, rows, width, max(sum(prompts), rows), dev)
        search = pkg("integration.beam").BeamSearch(tables, ops.PageSet(cache.planes()), beams, eos)

        def forward(tokens, t):
            n = tokens.numel()
            q, k, v = model.qkv(tokens, t.positions[:n])
            m = meta((t.slot_mapping[:n], t.query_start_loc), tables.block_table, t.seq_lens)
            return (impl.forward(None, q, k, v, cache, m).double() @ head).float()

        t = tables.step(lens)
        logits = forward(feed, t)[search.last_rows(t)]
        if not host:
            torch.cuda.set_sync_debug_mode("error")  # the loop waits for nothing
        for _ in range(steps):
            tokens = search.step(logits)
            t = tables.step(search.query_lens())
            if host:
                live = [r for r, d in enumerate(search.done.tolist()) if not d]
                if not live:
                    break
                packed = forward(tokens[live], t)
                logits = torch.zeros((rows, packed.shape[1]), device=dev)
                logits[live] = packed
            else:
                logits = forward(search.packed_tokens(), t)[search.last_rows(t)]
        return search

    try:
        a = run(False)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    b = run(True)
    assert eos < 0 or b.done.any()
    n = b.sequences().shape[2]
    assert torch.equal(a.sequences()[:, :, :n], b.sequences()) and not a.sequences()[:, :, n:].any()
    torch.testing.assert_close(a.scores, b.scores, rtol=1e-6, atol=1e-6)
    assert torch.equal(a.done, b.done)
