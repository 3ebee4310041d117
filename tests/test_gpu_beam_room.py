"""Beam search in a pool that runs out of pages: no beam goes on from logits of tokens that the
cache does not hold, and beams that have ended leave their pages to the others."""
import math

import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu
BS, VOCAB = 32, 100


def _search(pages, prompt, beams, eos=-1):
    ops, tab = pkg("native.torch_ops"), pkg("integration.block_table")
    tables = tab.DeviceBlockTables(pages, BS, beams, 4, 64, "cuda")
    cache = ops.q4_kv_cache(pages, BS, 1, 64, "cuda")
    search = pkg("integration.beam").BeamSearch(tables, ops.PageSet(cache.planes()), beams, eos)
    _take(tables, [prompt] + [0] * (beams - 1))
    return tables, search


def _take(tables, lens):
    return tables.step(torch.tensor(lens, dtype=torch.int32, device="cuda"))


def _logits(*rows):
    """Rows of 0 but for {token: logit}."""
    x = torch.zeros((len(rows), VOCAB), device="cuda")
    for r, row in enumerate(rows):
        for t, v in row.items():
            x[r, t] = v
    return x


def test_a_beam_without_a_page_for_its_copy():
    """Two beams of a prompt that fills the pool with a last page that is not full: the second
    finds no page for its copy.  Its logits, however good, are not gone on from."""
    tables, search = _search(2, 40, 2)
    assert search.step(_logits({5: 9.0, 7: 8.0}, {})).tolist() == [5, 7]
    assert tables.lens.tolist() == [40, 32]
    tables.step(search.query_lens())
    tokens = search.step(_logits({11: 3.0, 12: 2.0}, {13: 50.0}))
    assert tokens.tolist() == [11, 12]
    assert search.sequences().tolist() == [[[5, 11], [5, 12]]]
    assert torch.isfinite(search.scores).all()


def test_a_beam_without_a_page_for_its_token():
    """A full page and no other: the token that was taken is nowhere, and the search ends."""
    tables, search = _search(1, 32, 1)
    assert search.step(_logits({5: 9.0})).tolist() == [5]
    tables.step(search.query_lens())
    assert tables.lens.tolist() == [32]
    assert search.step(_logits({6: 9.0})).tolist() == [0]
    assert search.scores.tolist() == [[-math.inf]] and search.query_lens().tolist() == [0]
    # (and stays so)
    tables.step(search.query_lens())
    assert search.step(_logits({6: 9.0})).tolist() == [0]
    assert search.scores.tolist() == [[-math.inf]]


def test_an_ended_beam_gives_up_its_pages():
    """The beam that ends is the first child of its parent, the other takes the last page as it
    is: no copy is needed, and the search goes on where no other page is left."""
    tables, search = _search(2, 40, 2, eos=5)
    assert search.step(_logits({5: 9.0, 7: 8.0}, {})).tolist() == [5, 7]
    assert tables.lens.tolist() == [0, 40] and tables.num_pages.tolist() == [0, 2]
    own = search.scores[0, 0].item()
    for t in range(8, 14):
        held = tables.lens.tolist()[1]
        tables.step(search.query_lens())
        assert tables.lens.tolist() == [0, held + 1]
        search.step(_logits({}, {t: 60.0}))
        assert search.scores[0, 0].item() == own
    assert search.sequences().tolist() == [[[5, 0, 0, 0, 0, 0, 0], [7, 8, 9, 10, 11, 12, 13]]]


def test_the_room_that_ended_beams_leave_is_used():
    """Four beams of a pool that is just enough for one more page: ended ones' pages are taken
    by the others' copies a step later."""
    tables, search = _search(3, 33, 4, eos=1)
    search.step(_logits({5: 9.0, 1: 8.5, 6: 8.0, 7: 7.0}, {}, {}, {}))
    # rows 0 (5), 2 (6) and 3 (7) go on: one keeps the last page, one has the copy
    assert tables.lens.tolist() == [33, 0, 33, 32]
    tables.step(search.query_lens())
    search.step(_logits({1: 90.0}, {}, {8: 60.0, 9: 59.0}, {10: 99.0}))
    # row 3 is out; row 0 has ended, and its page is free for the next copy
    assert [s[-1] for s in search.sequences().view(4, -1).tolist()].count(10) == 0
    assert int(tables.free_count) + len({p for r, c in zip(
        tables.block_table.tolist(), tables.num_pages.tolist()) for p in r[:c]}) == 3
