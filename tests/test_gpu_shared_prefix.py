"""Decode attention of a batch that shares a prefix
(torch_ops.shared_prefix_attention), against float64 attention on the CPU."""
import math

import pytest
import torch

from _rows import assert_rows, prefix64
from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ops():
    return pkg("native.torch_ops")


def _case(seed, prefix, suffix, n_q, n_kv, hd, bs, own_prefix_entries=True):
    g = torch.Generator().manual_seed(seed)
    S = len(suffix)
    shared, pre = prefix // bs, -(-prefix // bs)
    per = max(-(-(prefix + max(suffix)) // bs), 1)
    blocks = max(pre, 1) + S * (per - shared) + 2
    k, v = (torch.randn((blocks, bs, n_kv, hd), generator=g).to(BF16) for _ in range(2))
    q = torch.randn((S, n_q, hd), generator=g).to(BF16)
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    ptable = perm[:max(pre, 1)].contiguous()
    tail = perm[max(pre, 1):max(pre, 1) + S * (per - shared)].view(S, per - shared)
    head = ptable[:shared].expand(S, shared) if own_prefix_entries else torch.full(
        (S, shared), -1, dtype=torch.int32)
    table = torch.cat((head, tail), 1).to(torch.int32).contiguous()
    lens = torch.tensor([prefix + x for x in suffix], dtype=torch.int32)
    return q, k, v, ptable, torch.tensor([prefix], dtype=torch.int32), table, lens


def _run(case, scale=0.1, **kw):
    return _ops().shared_prefix_attention(*[x.cuda() for x in case], scale, **kw)


def _check(case, scale=0.1, what=""):
    q, k, v, ptable, plen, table, lens = case
    ref, mag = prefix64(q, k, v, ptable, int(plen), table, lens, scale)
    assert_rows(_run(case, scale), ref, mag, what)


CASES = [
    # prefix, suffix lengths, n_q, n_kv, hd, bs
    (128, [1], 32, 8, 128, 128),
    (128, [1, 2, 3], 32, 8, 128, 128),
    (300, [1, 90, 7], 16, 4, 64, 64),
    (45, [5, 1, 64, 19], 8, 2, 128, 32),
    (1, [1, 1], 4, 1, 128, 32),
    (700, [0, 3, 0], 8, 8, 64, 32),
    (1000, [33, 500, 1, 129, 64], 10, 2, 128, 256),
    (257, [(5 * i) % 37 for i in range(40)], 14, 2, 64, 32),
    (640, [4, 70], 64, 1, 64, 32),
    (90, [200, 11], 100, 1, 64, 64),
    (2050, [1] * 16, 32, 8, 128, 128),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("entries", [True, False])
def test_matches_float64(case, entries):
    """With the prefix's pages in the sequences' own rows, and with -1 there."""
    print(f"prefix case {case} {entries}", flush=True)
    _check(_case(1, *case, own_prefix_entries=entries), what=str(case))


@pytest.mark.parametrize("seqs,prefix", [(64, 70), (70, 333), (130, 40), (100, 3900)])
def test_many_sequences(seqs, prefix):
    """More segments than one round of the search for a workgroup's item holds, with
    one list of them and with workgroups of the prefix's own (100 under 3900)."""
    suffix = [(37 * i) % 90 for i in range(seqs)]
    _check(_case(12, prefix, suffix, 8, 2, 64, 32), what=f"{seqs} under {prefix}")


def test_agrees_with_split_kv_decode():
    """The framework's decode attention over the same whole sequences: two
    evaluations of one function, each within the derived bound of it."""
    case = _case(2, 512, [3, 100, 40], 32, 8, 128, 128)
    q, k, v, ptable, plen, table, lens = [x.cuda() for x in case]
    ops = _ops()
    po, pl = ops.splitkv_decode(q, k, v, table, lens, 4, 0.1)
    ref, mag = prefix64(*case[:4], 512, *case[5:], 0.1)
    assert_rows(ops.lse_merge(po, pl), ref, mag, "split-KV")
    assert_rows(_run(case), ref, mag, "shared prefix")


def test_lengths_below_the_prefix_and_empty_rows():
    case = _case(3, 200, [5, 5, 5, 5], 8, 2, 128, 32)
    lens = case[6]
    lens[0], lens[1], lens[2] = 77, 0, -3
    got = _run(case).cpu()
    assert torch.equal(got[1:3], torch.zeros_like(got[1:3]))
    _check(case, what="short rows")


def test_no_prefix_and_a_prefix_past_its_table():
    case = list(_case(4, 64, [50, 9], 8, 2, 128, 32))
    case[4] = torch.tensor([0], dtype=torch.int32)
    case[5][:, :2] = case[3][:2]
    _check(case, what="prefix_len 0")
    case[4] = torch.tensor([-7], dtype=torch.int32)
    _check(case, what="prefix_len below 0")
    case[4] = torch.tensor([1000], dtype=torch.int32)  # the prefix table has 64 tokens
    _check(case, what="prefix_len past the table")


@pytest.mark.parametrize("seqs", [3, 40])
def test_a_prefix_longer_than_the_own_tables(seqs):
    """All sequences end within the prefix, whose last page is past their tables'."""
    q, k, v, ptable, plen, table, lens = _case(11, 3000, [1] * seqs, 8, 2, 128, 32)
    table = table[:, :4].contiguous()
    lens = torch.arange(seqs, dtype=torch.int32) * 7 % 129
    _check((q, k, v, ptable, plen, table, lens), what="narrow tables")


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_what_a_row_does_not_see_does_not_reach_it(bad):
    """Behind every sequence's end, behind the prefix's end in its last page, and in
    the own pages' slots below the prefix's end."""
    case = _case(5, 75, [30, 4, 90], 8, 2, 128, 32)
    q, k, v, ptable, plen, table, lens = case
    ref, mag = prefix64(q, k, v, ptable, 75, table, lens, 0.1)
    for c in (k, v):
        c[ptable[2], 75 % 32:] = bad
        for r in range(3):
            c[table[r, 2], :75 % 32] = bad
            for t in range(int(lens[r]), table.shape[1] * 32):
                c[table[r, t // 32], t % 32] = bad
    assert_rows(_run(case), ref, mag, f"{bad}")


def test_an_infinite_value_of_one_sequence_stays_there():
    case = _case(6, 64, [30, 4, 90], 8, 2, 128, 32)
    q, k, v, ptable, plen, table, lens = case
    ref, mag = prefix64(q, k, v, ptable, 64, table, lens, 0.1)
    v[table[0, 2], 3, 0, 11] = math.inf
    got = _run(case).cpu()
    assert (got[0, :4, 11].float() == math.inf).all()
    ref[0, :4, 11], mag[0, :4, 11], got[0, :4, 11] = 0, 0, 0
    assert_rows(got, ref, mag, "others")


@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_bad_pages(entry):
    case = _case(7, 96, [30, 4, 50], 8, 2, 128, 32)
    q, k, v, ptable, plen, table, lens = case
    ref, mag = prefix64(q, k, v, ptable, 96, table, lens, 0.1)
    table[1, 3] = entry
    got = _run(case).cpu()
    assert torch.isnan(got[1]).all()
    assert_rows(got[[0, 2]], ref[[0, 2]], mag[[0, 2]], "others")
    ptable[1] = entry
    assert torch.isnan(_run(case)).all()


def test_strided_queries_and_out():
    case = _case(8, 130, [3, 9, 70], 8, 2, 128, 64)
    wide = torch.randn((3, 12 * 128)).to(BF16).cuda()
    view = wide[:, :8 * 128].view(3, 8, 128)
    view.copy_(case[0])
    dev = [x.cuda() for x in case[1:]]
    out = torch.empty((3, 8, 128), dtype=BF16, device="cuda")
    a = _ops().shared_prefix_attention(view, *dev, 0.1, out=out)
    assert a is out
    assert torch.equal(a.view(torch.int16), _run(case).view(torch.int16))


def test_captured_and_replayed():
    case = [x.cuda() for x in _case(9, 300, [50, 9, 200], 32, 8, 128, 128)]
    ops = _ops()
    ws = ops.shared_prefix_attention_workspace(case[0], case[1], case[3], case[5])
    out = torch.empty_like(case[0])
    call = lambda: ops.shared_prefix_attention(*case, 0.1, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        case[4].sub_(40 * i)  # a shorter prefix: the rest is read from the own pages
        case[6].sub_(3)
        case[0].mul_(-1)
        for r in range(3):
            case[5][r, :2] = case[3][:2]
        ref = ops.shared_prefix_attention(*case, 0.1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), ref.view(torch.int16)), f"replay {i}"


def test_wrapper_refusals():
    ops = _ops()
    q, k, v, ptable, plen, table, lens = [x.cuda() for x in _case(10, 64, [3, 9], 8, 2, 128, 32)]
    ok = dict(q=q, k_cache=k, v_cache=v, prefix_table=ptable, prefix_len=plen, block_table=table,
              seq_lens=lens, scale=0.1)
    for change in (dict(q=q[:1].contiguous()), dict(prefix_table=ptable.long()),
                   dict(prefix_table=ptable.view(1, -1)), dict(prefix_len=plen.long()),
                   dict(prefix_len=plen.repeat(2)), dict(block_table=table.cpu()),
                   dict(prefix_table=ptable[:0])):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(**{**ok, **change})
    with pytest.raises(pkg("native").SmxError):
        ops.shared_prefix_attention(**{**ok, "workspace": torch.empty(16, dtype=torch.uint8,
                                                                      device="cuda")})
