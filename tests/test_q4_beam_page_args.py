"""CPU checks of the C entries of the 4-bit cache, the beam selection and the page
operators: bad arguments are refused on the host before anything is launched (the
pointers below are never dereferenced), and workspace sizes.  And the host restatements
that the GPU tests compare with, on cases worked out by hand."""
import math

import numpy as np
import pytest

from _pages import compact, fork
from _util import pkg
from oracle import q4_kv

W = dict(key=16, key_stride=1024, value=16, value_stride=1024, codes=16, scales=16, slots=16,
         tokens=4, n_kv=8, hd=128, num_blocks=9, bs=128)
N = dict(qkv=16, qg=16, kg=16, cs=16, pos=16, slots=16, q=16, codes=16, scales=16, tokens=4,
         n_q=32, n_kv=8, hd=128, num_blocks=9, bs=128, max_pos=100, eps=1e-6)
R = dict(codes=16, scales=16, slots=16, key=16, value=16, tokens=4, n_kv=8, hd=128,
         num_blocks=9, bs=128)
A = dict(q=16, q_stride=4096, codes=16, scales=16, table=16, start=16, lens=16, ws=16,
         ws_bytes=1 << 40, out=16, tokens=5, seqs=2, max_blocks=40, num_blocks=9, bs=128, n_q=32,
         n_kv=8, hd=128, scale=0.1)
B = dict(logits=16, stride=1000, size=2, scores=16, done=16, ws=16, ws_bytes=1 << 40, parents=16,
         tokens=16, out=32, seqs=2, beams=4, width=8, vocab=1000, pad=0)
F = dict(parents=1 << 20, lens=2 << 20, pages=3 << 20, free=4 << 20, count=5 << 20,
         table=6 << 20, table_out=7 << 20, pages_out=8 << 20, lens_out=9 << 20,
         free_out=10 << 20, count_out=11 << 20, copies=12 << 20, rows=8, max_blocks=4,
         num_blocks=90, num_free=90, bs=16)
C = dict(pages=16, table=1 << 20, table_out=2 << 20, free=16, count=16, moves=16, rows=8,
         max_blocks=4, num_blocks=90)
P = dict(planes=16, n=2, bytes=4096, pairs=16, num_pairs=3, num_blocks=9)

CACHE = [dict(codes=None), dict(scales=None), dict(codes=24), dict(scales=8), dict(tokens=0),
         dict(tokens=1 << 24), dict(n_kv=0), dict(hd=96), dict(hd=256), dict(num_blocks=0),
         dict(bs=16), dict(bs=96), dict(bs=8192), dict(slots=None), dict(slots=20)]


def _refused(name, base, change):
    native = pkg("native")
    lib = native.load()
    rc = getattr(lib, name)(None, *{**base, **change}.values())
    assert rc == native.SMX_EINVAL, change
    assert lib.smx_last_error().decode().startswith(name)


@pytest.mark.parametrize("change", CACHE + [
    dict(key=None), dict(value=None), dict(key=24), dict(value=8), dict(key_stride=1020),
    dict(key_stride=1028), dict(value_stride=512)], ids=str)
def test_write_refuses(change):
    _refused("smx_q4_reshape_and_cache", W, change)


@pytest.mark.parametrize("change", CACHE + [
    dict(qkv=None), dict(q=None), dict(cs=None), dict(pos=None), dict(pos=20), dict(qkv=24),
    dict(qg=8), dict(hd=64), dict(n_q=0), dict(n_q=70000), dict(tokens=65536), dict(max_pos=0),
    dict(eps=-1.0), dict(eps=math.nan), dict(tokens=65535, n_q=5000)], ids=str)
def test_norm_rope_write_refuses(change):
    _refused("smx_q4_qknorm_rope_kv_write", N, change)


@pytest.mark.parametrize("change", CACHE + [dict(key=None), dict(value=24)], ids=str)
def test_read_refuses(change):
    _refused("smx_q4_kv_read", R, change)


@pytest.mark.parametrize("change", [
    dict(q=None), dict(codes=None), dict(scales=None), dict(table=None), dict(lens=None),
    dict(out=None), dict(q=24), dict(codes=8), dict(scales=24), dict(out=24), dict(table=18),
    dict(lens=17), dict(start=18), dict(start=None), dict(q_stride=4088), dict(q_stride=4100),
    dict(seqs=0), dict(seqs=1 << 17), dict(tokens=0), dict(tokens=1 << 26), dict(max_blocks=0),
    dict(max_blocks=1 << 24), dict(num_blocks=0), dict(bs=96), dict(bs=16), dict(bs=8192),
    dict(n_q=33), dict(n_q=4), dict(n_kv=0), dict(hd=96), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=math.inf), dict(scale=math.nan), dict(n_q=1 << 17, n_kv=1 << 17), dict(ws=None),
    dict(ws=24), dict(ws_bytes=64), dict(tokens=1 << 21, q_stride=1 << 20, n_q=256, n_kv=1)],
    ids=str)
def test_attention_refuses(change):
    _refused("smx_q4_attention", A, change)


@pytest.mark.parametrize("change", [{k: None} for k in ("logits", "scores", "ws", "parents",
                                                        "tokens", "out")] + [
    dict(size=1), dict(size=8), dict(beams=0), dict(beams=65), dict(width=0), dict(width=65),
    dict(vocab=0), dict(vocab=(1 << 24) + 1, stride=1 << 25), dict(seqs=0), dict(seqs=20000),
    dict(stride=999), dict(pad=-1), dict(pad=1000), dict(logits=17), dict(logits=18, size=4),
    dict(ws=24), dict(scores=18), dict(parents=18), dict(tokens=20), dict(out=34),
    dict(out=16), dict(ws_bytes=99)], ids=str)
def test_beam_select_refuses(change):
    _refused("smx_beam_select", B, change)


@pytest.mark.parametrize("change", [{k: None} for k in list(F)[:12]] + [
    dict(rows=0), dict(rows=8193), dict(max_blocks=0), dict(max_blocks=1 << 28),
    dict(num_blocks=0), dict(num_blocks=(1 << 18) + 1), dict(num_free=0), dict(bs=0), dict(bs=24),
    dict(bs=8192), dict(parents=18), dict(copies=(12 << 20) + 2), dict(table_out=6 << 20),
    dict(table_out=(6 << 20) + 64), dict(pages_out=3 << 20), dict(pages_out=2 << 20),
    dict(lens_out=2 << 20), dict(lens_out=(1 << 20) + 28), dict(free_out=(4 << 20) + 40)], ids=str)
def test_fork_pages_refuses(change):
    _refused("smx_fork_pages", F, change)


@pytest.mark.parametrize("change", [{k: None} for k in list(C)[:6]] + [
    dict(rows=0), dict(rows=8193), dict(max_blocks=0), dict(num_blocks=0),
    dict(num_blocks=(1 << 18) + 1), dict(pages=18), dict(table_out=(1 << 20) + 16)], ids=str)
def test_compact_pages_refuses(change):
    _refused("smx_compact_pages", C, change)


@pytest.mark.parametrize("change", [
    dict(planes=None), dict(pairs=None), dict(planes=20), dict(pairs=18), dict(n=0),
    dict(n=65536), dict(bytes=8), dict(bytes=1 << 32), dict(num_pairs=0),
    dict(num_pairs=(1 << 18) + 1), dict(num_blocks=0)], ids=str)
def test_copy_pages_refuses(change):
    _refused("smx_copy_pages", P, change)


def test_workspace_sizes():
    lib = pkg("native").load()
    for bad in ((0, 1, 1, 32, 4, 1, 64), (1, 0, 1, 32, 4, 1, 64), (1, 1, 0, 32, 4, 1, 64),
                (1, 1, 1, 32, 5, 2, 64)):
        assert lib.smx_q4_attention_workspace(*bad) == -1
    assert lib.smx_q4_attention_workspace(4096, 1, 32, 128, 32, 8, 128) == 0
    assert lib.smx_q4_attention_workspace(1, 1, 256, 128, 32, 8, 128) > 0
    for bad in ((0, 1, 1, 9, 2), (1, 0, 1, 9, 2), (1, 1, 0, 9, 2), (1, 1, 1, 0, 2), (1, 1, 1, 9, 1)):
        assert lib.smx_beam_select_workspace(*bad) == -1
    assert lib.smx_beam_select_workspace(1, 1, 1, 1, 2) > 0


def test_quantisation_by_hand():
    x = np.zeros((1, 32))
    x[0, :6] = [-8.0, 7.0, 0.5, 0.49, -0.5, 8.0]
    c, d = q4_kv.quantise(x)
    assert d[0, 0] == 1.0  # -8 is the first of the largest
    assert c[0, :7].tolist() == [0, 15, 9, 8, 8, 15, 8]
    assert q4_kv.values(c, d)[0, :6].tolist() == [-8.0, 7.0, 1.0, 0.0, 0.0, 7.0]
    for hd in (64, 128):
        assert sorted(q4_kv.key_order(hd)) == list(range(hd))
        c = np.random.default_rng(1).integers(0, 16, (3, hd))
        for key in (True, False):
            assert (q4_kv.unpack(q4_kv.pack(c, key), key) == c).all()
    # dword 1 of a K row of 128: block 1's first eight channels, the even ones first
    assert q4_kv.key_order(128)[8:16] == [32, 34, 36, 38, 33, 35, 37, 39]
    # dword 4: block 0's next eight
    assert q4_kv.key_order(128)[32:36] == [8, 10, 12, 14]


def test_fork_by_hand():
    # two beams of 5 tokens (pages of 4) that share page 7; both go on with the second
    out = fork([1, 1], [5, 5], [2, 2], [3, 9], [[7, 1, -1], [7, 2, -1]], 10, 4)
    assert out == ([[7, 2, -1], [7, 9, -1]], [2, 2], [5, 5], [3, 1], [[-1, -1], [2, 9]])
    # whole pages are shared and not copied
    out = fork([0, 0], [4, 0], [1, 0], [3], [[7, -1], [-1, -1]], 10, 4)
    assert out == ([[7, -1], [7, -1]], [1, 1], [4, 4], [3], [[-1, -1], [-1, -1]])


def test_compact_by_hand():
    out = compact([2, 1], [[5, 0, 3], [2, -1, -1]], 6)
    assert out == ([[1, 0, -1], [2, -1, -1]], [5, 4, 3], [[5, 1]])
