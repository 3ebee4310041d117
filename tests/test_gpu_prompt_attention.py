"""Causal attention of packed query rows over the paged cache
(torch_ops.prompt_attention), against float64 attention on the CPU."""
import math

import pytest
import torch

from _rows import assert_rows, prompt64
from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ops():
    return pkg("native.torch_ops")


def _case(seed, n, ctx, n_q, n_kv, hd, bs, pad=0, spare=1, blocks_more=3):
    """Random inputs on the CPU: q [sum n + pad, n_q, hd], caches, table, start, lens."""
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(n, ctx)]
    per = -(-max(max(lens), 1) // bs) + spare
    blocks = len(n) * per + blocks_more
    k, v = (torch.randn((blocks, bs, n_kv, hd), generator=g).to(BF16) for _ in range(2))
    q = torch.randn((sum(n) + pad, n_q, hd), generator=g).to(BF16)
    table = torch.randperm(blocks, generator=g)[:len(n) * per].to(torch.int32).view(len(n), per)
    start = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32)
    return q, k, v, table, start, torch.tensor(lens, dtype=torch.int32)


def _run(q, k, v, table, start, lens, scale, **kw):
    dev = [x.cuda() for x in (q, k, v, table, start, lens)]
    return _ops().prompt_attention(*dev, scale, **kw)


CASES = [
    # n, ctx, n_q, n_kv, hd, bs, pad
    ([1], [0], 4, 1, 128, 32, 0),
    ([1], [0], 32, 8, 128, 128, 0),
    ([17], [0], 32, 8, 128, 128, 0),
    ([64], [0], 4, 2, 64, 64, 0),
    ([33, 1, 0, 65, 2], [0, 0, 0, 0, 0], 8, 2, 128, 32, 7),
    ([0, 0, 5], [3, 0, 1], 6, 6, 64, 32, 1),
    ([200], [0], 14, 2, 64, 32, 0),
    ([130], [71], 10, 2, 128, 64, 0),
    ([5, 5, 5], [100, 641, 1003], 32, 8, 128, 128, 0),
    ([1, 1, 1, 1], [0, 31, 32, 900], 32, 8, 128, 128, 2),
    ([3], [2000], 8, 1, 128, 256, 0),
    ([300], [0], 3, 1, 128, 4096, 0),
    ([77, 130], [64, 0], 40, 8, 128, 128, 0),
    ([257], [0], 64, 1, 64, 32, 0),
    ([9], [500], 100, 1, 64, 64, 0),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_matches_float64(case):
    n, ctx, n_q, n_kv, hd, bs, pad = case
    print(f"prompt case {case}", flush=True)
    q, k, v, table, start, lens = _case(1, n, ctx, n_q, n_kv, hd, bs, pad)
    out = torch.full(q.shape, 7.0, dtype=BF16, device="cuda")
    got = _run(q, k, v, table, start, lens, 1 / math.sqrt(hd), out=out)
    assert got is out
    ref, mag, mine = prompt64(q, k, v, table, start, lens, 1 / math.sqrt(hd))
    got = got.cpu()
    assert torch.equal(got[~mine], torch.full_like(got[~mine], 7.0)), "rows of no sequence"
    assert_rows(got[mine], ref[mine], mag[mine], str(case))


@pytest.mark.parametrize("n,ctx,n_q,n_kv,spare", [
    ([200], [0], 16, 4, 90), ([5, 3], [10, 3000], 32, 8, 60), ([1] * 22, [700] * 22, 8, 8, 60),
    ([1] * 22, [700] * 21 + [2100], 8, 8, 60), ([30, 400], [5000, 2], 8, 1, 0),
    ([300], [9000], 8, 2, 0), ([70, 90, 128], [0, 3, 0], 128, 32, 1)])
def test_lengths_far_below_the_capacity_and_uneven(n, ctx, n_q, n_kv, spare):
    """Both sides of the rules that cut a tile's tokens: by the tables' capacity on
    the host, by the lengths on the device (heads of 64, 128 tokens a page)."""
    case = _case(16, n, ctx, n_q, n_kv, 64, 128, spare=spare)
    print(n, ctx, flush=True)
    assert_rows(_run(*case, 0.1), *prompt64(*case, 0.1)[:2], f"{n} {ctx}")


def test_one_capture_cuts_and_does_not():
    """One captured call whose replays take whole tiles and cut ones in turn: what the
    other form left in the workspace does not matter."""
    q, k, v, table, start, lens = [x.cuda() for x in _case(17, [24], [5000], 8, 2, 128, 64)]
    ops = _ops()
    ws = ops.prompt_attention_workspace(q, k, table)
    assert ws is not None
    ws.fill_(255)
    out = torch.empty_like(q)
    call = lambda: ops.prompt_attention(q, k, v, table, start, lens, 0.1, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    cpu = [x.cpu() for x in (q, k, v, table, start)]
    for length in (100, 5024, 24, 4000, 0, 300):
        lens.fill_(length)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        ref, mag, _ = prompt64(*cpu, torch.tensor([length], dtype=torch.int32), 0.1)
        assert_rows(out, ref, mag, f"length {length}")


def test_many_sequences():
    """More sequences than one round of the tile search, most of them tiny."""
    n = [(7 * i) % 5 for i in range(150)]
    ctx = [(13 * i) % 40 for i in range(150)]
    q, k, v, table, start, lens = _case(2, n, ctx, 4, 1, 64, 32, pad=3)
    got = _run(q, k, v, table, start, lens, 0.125)
    ref, mag, mine = prompt64(q, k, v, table, start, lens, 0.125)
    assert_rows(got.cpu()[mine], ref[mine], mag[mine], "150 sequences")


def test_rows_that_see_nothing_are_zero():
    """seq_lens below the number of query tokens (and 0): those tokens stand before
    the first position."""
    q, k, v, table, start, lens = _case(3, [40, 8, 3], [0, 0, 0], 8, 2, 128, 32)
    lens[0], lens[1], lens[2] = 33, 0, -5
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    ref, mag, _ = prompt64(q, k, v, table, start, lens, 0.1)
    assert torch.equal(got[:7], torch.zeros_like(got[:7]))
    assert torch.equal(got[40:], torch.zeros_like(got[40:]))
    assert_rows(got, ref, mag, "short lengths")


def test_length_past_the_table_counts_as_its_capacity():
    q, k, v, table, start, lens = _case(4, [5], [59], 4, 1, 128, 32, spare=0)
    lens[0] = 1000  # the table holds 64 tokens
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    ref, mag, _ = prompt64(q, k, v, table, start, lens, 0.1)
    assert_rows(got, ref, mag, "capacity")


def test_offsets_past_the_rows_are_clamped():
    q, k, v, table, start, lens = _case(5, [20, 9], [0, 0], 4, 1, 64, 32)
    start[2] = 500
    got = _run(q[:25].contiguous(), k, v, table, start, lens, 0.1).cpu()
    ref, mag, _ = prompt64(q[:25], k, v, table, start, lens, 0.1)
    assert_rows(got, ref, mag, "offsets")


@pytest.mark.parametrize("hd", [64, 128])
def test_strided_queries(hd):
    """q as the first heads of QKV rows, and the same values contiguous: the same bits."""
    q, k, v, table, start, lens = _case(6, [50, 3], [10, 90], 8, 2, hd, 64)
    wide = torch.randn((53, 12 * hd)).to(BF16).cuda()
    view = wide[:, :8 * hd].view(53, 8, hd)
    view.copy_(q)
    dev = [x.cuda() for x in (k, v, table, start, lens)]
    a = _ops().prompt_attention(view, *dev, 0.1)
    b = _ops().prompt_attention(q.cuda(), *dev, 0.1)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,ctx", [([100], [0]), ([4], [300]), ([40, 70], [0, 64])])
def test_what_a_row_does_not_see_does_not_reach_it(bad, n, ctx):
    """Unwritten slots behind a sequence's end, and K and V of later tokens, hold
    infinities and NaN: every row before them is as if they were not there."""
    q, k, v, table, start, lens = _case(7, n, ctx, 8, 2, 128, 64)
    ref, mag, _ = prompt64(q, k, v, table, start, lens, 0.1)
    tail = []
    for r in range(len(n)):
        L, bs = int(lens[r]), 64
        for t in range(L, table.shape[1] * bs):  # never written
            k[table[r, t // bs], t % bs] = bad
            v[table[r, t // bs], t % bs] = bad
        t = L - 2  # the last but one token: seen by the last two rows alone
        k[table[r, t // bs], t % bs, :, 3] = bad
        v[table[r, t // bs], t % bs, :, 5] = bad
        tail += [int(start[r + 1]) - 2, int(start[r + 1]) - 1]
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    keep = [i for i in range(q.shape[0]) if i not in tail]
    assert_rows(got[keep], ref[keep], mag[keep], f"{bad}")
    if not math.isnan(bad):  # K's values may give p = 0 or NaN there, V's alone reach dim 5
        return
    assert torch.isnan(got[tail]).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_a_row_sees_reaches_it(bad):
    """An infinite (NaN) V of a seen token gives an infinite (NaN) output in its dim
    and leaves the others; rows before it stay finite."""
    q, k, v, table, start, lens = _case(8, [90], [0], 4, 1, 128, 32)
    ref, mag, _ = prompt64(q, k, v, table, start, lens, 0.1)
    v[table[0, 70 // 32], 70 % 32, 0, 9] = bad
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    assert_rows(got[:70], ref[:70], mag[:70], "before")
    hit = got[70:, :, 9].float()
    assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
    rest = [d for d in range(128) if d != 9]
    assert_rows(got[70:][..., rest], ref[70:][..., rest], mag[70:][..., rest], "other dims")


@pytest.mark.parametrize("entry", [-1, 10 ** 6, -2 ** 31])
def test_bad_pages_give_nan_to_the_rows_that_see_them(entry):
    q, k, v, table, start, lens = _case(9, [100, 20], [0, 40], 8, 2, 128, 32)
    ref, mag, _ = prompt64(q, k, v, table, start, lens, 0.1)
    table[0, 1] = entry            # tokens 32..63 of sequence 0
    table[0, table.shape[1] - 1] = entry  # past every length: not seen
    table[1, table.shape[1] - 1] = entry
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    assert torch.isnan(got[32:100]).all()
    keep = list(range(32)) + list(range(100, 120))
    assert_rows(got[keep], ref[keep], mag[keep], f"entry {entry}")


def test_large_and_tiny_scores():
    """Scores to about 2000 (a softmax of one token) and a scale of 1e-6 (an average)."""
    for scale, mul in ((1.0, 12.0), (1e-6, 1.0)):
        q, k, v, table, start, lens = _case(10, [70], [60], 8, 2, 128, 64)
        k = k.float().mul(mul).to(BF16)
        got = _run(q, k, v, table, start, lens, scale).cpu()
        ref, mag, _ = prompt64(q, k, v, table, start, lens, scale)
        # fp32 scores of magnitude s are off by up to s * 2^-24 * 128 in the exponent
        mag = mag * (1 + (2.0 ** 11 * 128 * 2.0 ** -24 * 128 if mul > 1 else 0))
        assert_rows(got, ref, mag, f"scale {scale}")


def test_cache_offsets_past_32_bits():
    """Pages whose elements lie beyond 2^32 bytes and 2^31 elements."""
    n_kv, hd, bs = 8, 128, 128
    blocks = (2 ** 31 + 2 ** 24) // (n_kv * hd * bs)
    q, k, v, table, start, lens = _case(11, [40], [200], 16, n_kv, hd, bs, spare=0)
    big_k = torch.empty((blocks, bs, n_kv, hd), dtype=BF16, device="cuda")
    big_v = torch.empty_like(big_k)
    pages = torch.tensor([[blocks - 1, blocks - 3]], dtype=torch.int32)
    for i in range(2):
        big_k[pages[0, i]] = k[table[0, i]].cuda()
        big_v[pages[0, i]] = v[table[0, i]].cuda()
    got = _ops().prompt_attention(q.cuda(), big_k, big_v, pages.cuda(), start.cuda(),
                                  lens.cuda(), 0.1)
    ref, mag, _ = prompt64(q, k, v, table, start, lens, 0.1)
    assert_rows(got, ref, mag, "far pages")


@pytest.mark.parametrize("n,ctx", [([300, 41], [0, 100]), ([4, 3], [1500, 900])])
def test_captured_replayed_and_repeated(n, ctx):
    """A captured call replayed on new lengths, tables and rows, with eager calls of
    the same operator between: each replay equals the eager result bit for bit."""
    q, k, v, table, start, lens = [x.cuda() for x in _case(12, n, ctx, 8, 2, 128, 64)]
    ops = _ops()
    ws = ops.prompt_attention_workspace(q, k, table)
    out = torch.empty_like(q)
    call = lambda: ops.prompt_attention(q, k, v, table, start, lens, 0.1, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        lens.sub_(7 * i)
        q.mul_(-1)
        ref = ops.prompt_attention(q, k, v, table, start, lens, 0.1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), ref.view(torch.int16)), f"replay {i}"


def test_two_streams_at_once():
    """Calls on two streams with workspaces of their own, against one after the other."""
    ops = _ops()
    cases = [[x.cuda() for x in _case(s, [3, 9], [1800, 700], 32, 8, 128, 128)] for s in (13, 14)]
    want = [ops.prompt_attention(*c, 0.1) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.prompt_attention(*cases[i], 0.1)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_wrapper_refusals():
    ops = _ops()
    q, k, v, table, start, lens = [x.cuda() for x in _case(15, [5], [3], 8, 2, 128, 32)]
    ok = dict(q=q, k_cache=k, v_cache=v, block_table=table, query_start_loc=start, seq_lens=lens,
              scale=0.1)
    bad = [dict(q=q.float()), dict(q=q[:, :, ::2]), dict(q=q.cpu()), dict(q=q[0]),
           dict(k_cache=k[:, :, :, :64]), dict(v_cache=v[1:]), dict(v_cache=v.half()),
           dict(block_table=table.long()), dict(block_table=table[0]),
           dict(query_start_loc=start[:1]), dict(query_start_loc=start.long()),
           dict(seq_lens=lens.repeat(2)), dict(out=q[:3].clone()),
           dict(q=torch.empty((5, 8 * 128 + 4), dtype=BF16, device="cuda")[:, 4:].view(5, 8, 128)),
           dict(workspace=torch.empty(4, device="cuda"))]
    for change in bad:
        with pytest.raises((ValueError, RuntimeError)):
            ops.prompt_attention(**{**ok, **change})
    for change in (dict(scale=0.0), dict(scale=math.inf), dict(q=q[:, :7].contiguous())):
        with pytest.raises(pkg("native").SmxError):
            ops.prompt_attention(**{**ok, **change})
