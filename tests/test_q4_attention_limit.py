"""The most work that a call of the attention over a cache in 4 bits takes: row tiles of 16
times the tables' capacity in rounds of 128 tokens, refused on the host from 2^28 on (the
pointers below are never dereferenced)."""
import pytest

from _util import pkg


@pytest.mark.parametrize("seqs,max_blocks,bs", [(128, 1 << 16, 4096), (65535, 4097, 128),
                                                (16384, 16384, 128)])
def test_the_most_work(seqs, max_blocks, bs):
    assert seqs * max_blocks * bs // 128 >= 1 << 28
    native = pkg("native")
    lib = native.load()
    rc = lib.smx_q4_attention(None, 16, 128, 16, 16, 16, None, 16, 16, 1 << 40, 16, seqs, seqs,
                              max_blocks, 9, bs, 1, 1, 128, 0.1)
    assert rc == native.SMX_EINVAL
    said = lib.smx_last_error().decode()
    assert "capacity / 128" in said and "2^28" in said
