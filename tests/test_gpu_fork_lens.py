"""DeviceBlockTables.fork with lengths: rows that share pages are taken back to fewer tokens, as
drafted ones that were not accepted are, where keep() is refused."""
import numpy as np
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu
BS = 32


def test_rows_are_taken_back_after_a_fork():
    """Against what each row's tokens are: written by their number into pages, and followed
    through forks that shorten the rows, with the copies that they ask for."""
    ops, tab = pkg("native.torch_ops"), pkg("integration.block_table")
    rows, blocks, width = 4, 40, 8
    i32 = dict(dtype=torch.int32, device="cuda")
    t = tab.DeviceBlockTables(blocks, BS, rows, width, 300, "cuda")
    pool = torch.zeros((1, blocks, BS, 4), **i32)
    pages = ops.PageSet([pool])
    rng = np.random.default_rng(2)
    texts, count = [[] for _ in range(rows)], 0
    for turn in range(40):
        takes = rng.integers(0, 45, rows)
        takes = [int(min(n, width * BS - len(x))) for n, x in zip(takes, texts)]
        step = t.step(torch.tensor(takes, **i32))
        slots = step.slot_mapping[:sum(takes)].cpu()
        new = list(range(count, count + sum(takes)))
        count += sum(takes)
        pool.view(-1, 4)[slots[slots >= 0].cuda(), 0] = torch.tensor(new, **i32)[(slots >= 0).cuda()]
        at = 0
        for r, n in enumerate(takes):
            kept = [x for x, s in zip(new[at:at + n], slots[at:at + n].tolist()) if s >= 0]
            texts[r] = texts[r] + kept
            at += n
        assert t.lens.tolist() == [len(x) for x in texts]
        parents = rng.integers(-1, rows, rows)
        if turn % 3 == 0:
            parents = np.arange(rows)
        keep = rng.integers(-3, width * BS + 3, rows) if turn % 4 else np.array(
            [max(len(x) - 3, 0) for x in texts])
        ops.copy_pages(pages, t.fork(torch.tensor(parents, **i32), torch.tensor(keep, **i32)))
        want = [texts[p][:max(int(keep[p]), 0)] if p >= 0 else [] for p in parents]
        lens = t.lens.tolist()
        for r in range(rows):  # (a row whose copy found no page is cut to whole pages)
            assert lens[r] == len(want[r]) or lens[r] == len(want[r]) // BS * BS
        texts = [x[:n] for x, n in zip(want, lens)]
        held = pool[0, :, :, 0].cpu()
        table = t.block_table.cpu()
        for r, x in enumerate(texts):
            n = len(x)
            assert torch.equal(held[table[r, :-(-n // BS)].long()].flatten()[:n],
                               torch.tensor(x, dtype=torch.int32)), (turn, r)
        listed = {p for r, c in zip(table.tolist(), t.num_pages.tolist()) for p in r[:c]}
        left = t.free_pages[:int(t.free_count)].tolist()
        assert sorted(listed | set(left)) == list(range(blocks)) and not listed & set(left)
    with pytest.raises(RuntimeError, match="lens"):
        t.keep(torch.zeros(rows, **i32))


def test_lens_must_be_the_tables():
    tab = pkg("integration.block_table")
    t = tab.DeviceBlockTables(8, BS, 2, 4, 64, "cuda")
    rows = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (rows.long(), rows[:1], torch.zeros(3, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="lens"):
            t.fork(rows, bad)
