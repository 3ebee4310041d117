"""CPU checks of the row attentions' and the request tables' C entries: bad
arguments are refused on the host before anything is launched (the pointers
below are never dereferenced), and workspace sizes."""
import math

import pytest

from _util import pkg

P = dict(q=16, q_stride=4096, k=16, v=16, table=16, start=16, lens=16, ws=16, ws_bytes=1 << 40,
         out=16, tokens=5, seqs=2, max_blocks=4, num_blocks=9, bs=128, n_q=32, n_kv=8, hd=128,
         scale=0.1)
S = dict(q=16, q_stride=4096, k=16, v=16, ptable=16, plen=16, table=16, lens=16, ws=16,
         ws_bytes=1 << 40, out=16, seqs=2, pblocks=3, max_blocks=4, num_blocks=9, bs=128, n_q=32,
         n_kv=8, hd=128, scale=0.1)
T = dict(query=16, context=32, pages=16, free=16, count=16, table=16, pages_out=16, count_out=16,
         start=16, lens=16, pos=16, slots=16, reqs=2, tokens=8, max_blocks=4, num_free=9, bs=16)
R = dict(keep=16, pages=16, free=16, count=16, table=16, reqs=2, max_blocks=4, num_free=9, bs=16)

SHARED = [dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lens=None),
          dict(out=None), dict(q=24), dict(k=8), dict(v=17), dict(out=24), dict(table=18),
          dict(lens=17), dict(q_stride=4088), dict(q_stride=4100), dict(seqs=0),
          dict(seqs=1 << 17), dict(max_blocks=0), dict(max_blocks=1 << 24), dict(num_blocks=0),
          dict(bs=96), dict(bs=16), dict(bs=8192), dict(n_q=33), dict(n_q=4), dict(n_kv=0),
          dict(hd=96), dict(hd=256), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf),
          dict(scale=math.nan), dict(n_q=1 << 17, n_kv=1 << 17)]


def _refused(name, base, change):
    native = pkg("native")
    lib = native.load()
    rc = getattr(lib, name)(None, *{**base, **change}.values())
    assert rc == native.SMX_EINVAL, change
    assert lib.smx_last_error().decode().startswith(name)


@pytest.mark.parametrize("change", SHARED + [dict(start=None), dict(start=18), dict(tokens=0),
                                             dict(tokens=1 << 26)], ids=str)
def test_prompt_attention_refuses(change):
    _refused("smx_prompt_attention", P, change)


@pytest.mark.parametrize("change", SHARED + [dict(ptable=None), dict(plen=None), dict(plen=17),
                                             dict(pblocks=0), dict(pblocks=1 << 24),
                                             dict(ws=None), dict(ws=24), dict(ws_bytes=64)],
                         ids=str)
def test_shared_prefix_attention_refuses(change):
    _refused("smx_shared_prefix_attention", S, change)


@pytest.mark.parametrize("change", [{k: None} for k in list(T)[:12]]
                         + [dict(query=18), dict(pos=20), dict(slots=12), dict(reqs=0),
                            dict(reqs=1 << 17), dict(tokens=0), dict(max_blocks=0),
                            dict(reqs=60000, max_blocks=1 << 20),
                            dict(reqs=1, max_blocks=2 ** 31 - 1), dict(num_free=0), dict(bs=0),
                            dict(bs=24), dict(bs=8192), dict(lens=32, query=32)], ids=str)
def test_request_tables_refuses(change):
    base = dict(T, lens=48)
    _refused("smx_request_tables", base, change)


@pytest.mark.parametrize("change", [{k: None} for k in list(R)[:5]]
                         + [dict(keep=18), dict(reqs=0), dict(max_blocks=0), dict(num_free=0),
                            dict(bs=24)], ids=str)
def test_release_pages_refuses(change):
    _refused("smx_release_pages", R, change)


def test_workspace_sizes():
    """None for prompts that fill the chip; partials of every split elsewhere; a bad
    size is -1."""
    lib = pkg("native").load()
    assert lib.smx_prompt_attention_workspace(8192, 1, 64, 128, 32, 8, 128) == 0
    for bad in ((0, 1, 1, 32, 4, 1, 64), (1, 0, 1, 32, 4, 1, 64), (1, 1, 0, 32, 4, 1, 64),
                (1, 1, 1, 32, 5, 2, 64)):
        assert lib.smx_prompt_attention_workspace(*bad) == -1
        assert lib.smx_shared_prefix_attention_workspace(*bad[:1], 1, *bad[2:]) == -1 or bad[1] == 0
    for seqs, hd in ((1, 128), (64, 64)):
        n = lib.smx_shared_prefix_attention_workspace(seqs, 256, 300, 128, 32, 8, hd)
        slots = (n / (seqs * 32 * 4) - 2) / (hd + 1)  # partials, lse, two counts a row
        assert n > 0 and slots == int(slots) >= 2
