"""Attention over a KV cache held in 4 bits (torch_ops.q4_attention) against float64
attention over the values that it holds."""
import math

import numpy as np
import pytest
import torch

from _rows import FP32, U, attend64
from _util import pkg
from oracle import q4_kv

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ops():
    return pkg("native.torch_ops")


class Case:
    """Random inputs on the CPU: q, a cache of N(0, 1) values, table, start, lens."""

    def __init__(self, seed, n, ctx, n_q, n_kv, hd, bs, pad=0, spare=1):
        g = torch.Generator().manual_seed(seed)
        lens = [a + b for a, b in zip(n, ctx)]
        per = -(-max(max(lens), 1) // bs) + spare
        blocks = len(n) * per + 3
        kv = torch.randn((2, blocks, n_kv, bs, hd), generator=g).to(BF16).float().numpy()
        cd = [q4_kv.quantise(kv[i]) for i in range(2)]
        self.codes = torch.from_numpy(np.stack([q4_kv.pack(c, i == 0)
                                                for i, (c, _) in enumerate(cd)]))
        self.scales = torch.from_numpy(np.stack([d for _, d in cd]))
        self.q = torch.randn((sum(n) + pad, n_q, hd), generator=g).to(BF16)
        self.table = torch.randperm(blocks, generator=g)[:len(n) * per].to(torch.int32).view(
            len(n), per)
        self.start = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.scale = 1 / math.sqrt(hd)

    def run(self, decode=False, **kw):
        q, codes, scales, table, lens, start = (x.cuda() for x in (
            self.q, self.codes, self.scales, self.table, self.lens, self.start))
        return _ops().q4_attention(q, _ops().Q4KVCache(codes, scales), table, lens, self.scale,
                                   query_start_loc=None if decode else start, **kw)

    def prompts(self):
        """Whether the rows go to the kernels that round the cache's values to bf16: more
        than 32 (token, head in the group) pairs a sequence on average, padding among them,
        and more than so many tiles of 16 of them times 128 tokens."""
        hd, n_kv, bs = self.q.shape[2], self.codes.shape[2], self.codes.shape[3]
        rows, seqs = self.q.shape[0] * (self.q.shape[1] // n_kv), len(self.lens)
        work = (-(-rows // 16) + seqs - 1) * (-(-self.table.shape[1] * bs // 128) + 3) * n_kv
        return rows > 32 * seqs and work > (9600 if hd == 64 else 5500)

    def reference(self):
        """(out, sum p |v|, sum p |d|, the largest scale sum |q k| of a seen token, row is of
        a sequence)"""
        codes, scales = self.codes.numpy(), self.scales.numpy()
        k, v = (torch.from_numpy(q4_kv.plane_values(codes, scales, i)) for i in range(2))
        d = torch.from_numpy(np.repeat(scales[1].astype(np.float64), 32, -1).transpose(0, 2, 1, 3))
        bs = k.shape[1]
        cap = self.table.shape[1] * bs
        out, mag, unit, top = (torch.zeros(self.q.shape, dtype=torch.float64) for _ in range(4))
        mine = torch.zeros(self.q.shape[0], dtype=torch.bool)
        for r in range(len(self.lens)):
            a, b = (min(int(self.start[r + i]), self.q.shape[0]) for i in range(2))
            if b <= a:
                continue
            mine[a:b] = True
            L = min(max(int(self.lens[r]), 0), cap)
            if L == 0:
                continue
            seen = torch.arange(L)[None] <= torch.arange(L - (b - a), L)[:, None]
            kk, vv, dd = (x[self.table[r, :-(-L // bs)].long()].flatten(0, 1)[:L]
                          for x in (k, v, d))
            out[a:b], mag[a:b] = attend64(self.q[a:b].double(), kk, vv, self.scale, seen)
            unit[a:b] = attend64(self.q[a:b].double(), kk, dd, self.scale, seen)[1]
            qk = torch.einsum("rhd,thd->rht", self.q[a:b].double().abs(), kk.abs()
                              .repeat_interleave(self.q.shape[1] // k.shape[2], 1)) * self.scale
            top[a:b] = torch.where(seen[:, None], qk, 0.0).amax(-1)[..., None]
        return out, mag, unit, top, mine

    def check(self, got, what="", rows=None):
        """The output's rounding to bf16 and the weights' (U), what fp32 adds to the scores
        (FP32; a score's products are of 16 + code, below 31, where _rows counts |v|, and
        sums of 32 in one instruction), and to sums of weights times 16 + code, up to 31
        times the weight's scale: one for every 32 tokens of a wave's quarter of them
        and 8 to join, half a step of fp32 (2^-24) doubled for the products inside.
        Prompts: V rounded to bf16 (U sum p |v|), and K, which moves every score by at most
        e = U scale sum |q k|, a weight p by p (exp(2 e) - 1) at most with the sum's change,
        and the output by that times (sum p |v| + |out|)."""
        ref, mag, unit, top, mine = self.reference()
        got = got.double().cpu()
        rows = mine if rows is None else rows
        assert torch.isfinite(got[rows]).all(), f"{what}: not finite"
        chain = int(self.lens.max().clamp(min=0)) / 32 + 8
        bound = (U * ref.abs() + (U + FP32) * mag + 31 * 2.0 ** -23 * chain * unit + 1e-30)
        if self.prompts():
            bound += U * mag + torch.expm1(2 * U * top) * (mag + ref.abs())
        over = ((got - ref).abs() / bound)[rows]
        worst = over.max().item() if over.numel() else 0.0
        assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


CASES = [
    # n, ctx, n_q, n_kv, hd, bs, pad
    ([1], [0], 4, 1, 128, 32, 0),
    ([1], [0], 1, 1, 64, 32, 0),
    ([1], [512], 32, 8, 128, 128, 0),
    ([1, 1, 1, 1], [0, 31, 63, 64], 32, 8, 128, 32, 0),
    ([1, 1, 1], [255, 256, 5000], 14, 2, 64, 64, 0),
    ([17], [0], 32, 8, 128, 128, 0),
    ([33, 1, 0, 65, 2], [0, 0, 0, 0, 0], 8, 2, 128, 32, 7),
    ([0, 0, 5], [3, 0, 1], 6, 6, 64, 32, 1),
    ([200], [0], 14, 2, 64, 32, 0),
    ([130], [71], 10, 2, 128, 64, 0),
    ([5, 5, 5], [100, 641, 1003], 32, 8, 128, 128, 0),
    ([1, 1, 1, 1], [0, 31, 32, 900], 32, 8, 128, 128, 2),
    ([3], [2000], 8, 1, 128, 256, 0),
    ([77, 130], [64, 0], 40, 8, 128, 128, 0),
    ([257], [0], 64, 1, 64, 32, 0),
    ([9], [500], 100, 1, 64, 64, 0),
    ([2], [300], 34, 2, 128, 4096, 0),
    # many rows: on both sides of what goes to the prompt kernels
    ([64, 100, 3], [0, 333, 900], 32, 8, 128, 32, 4),
    ([300], [0], 32, 8, 128, 64, 0),
    ([310, 77], [31, 500], 40, 8, 128, 128, 3),
    ([200, 1, 450], [64, 1000, 0], 16, 4, 64, 32, 0),
    ([500], [300], 28, 4, 64, 128, 2),
    ([40, 40, 40, 40, 0, 1], [700, 0, 50, 64, 0, 9], 64, 16, 64, 64, 0),
    ([1, 600], [0, 40], 16, 1, 128, 256, 0),
]


def test_cases_reach_both_kernels():
    kinds = {hd: {Case(1, n, ctx, n_q, n_kv, hd, bs, pad).prompts()
                  for n, ctx, n_q, n_kv, h, bs, pad in CASES if h == hd} for hd in (64, 128)}
    assert kinds == {64: {True, False}, 128: {True, False}}


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_matches_float64(case):
    n, ctx, n_q, n_kv, hd, bs, pad = case
    print(f"case {case}", flush=True)
    c = Case(1, n, ctx, n_q, n_kv, hd, bs, pad)
    out = torch.full(c.q.shape, 7.0, dtype=BF16, device="cuda")
    assert c.run(out=out) is out
    mine = c.reference()[4]
    assert torch.equal(out.cpu()[~mine], torch.full_like(c.q[~mine], 7.0)), "rows of no sequence"
    c.check(out, str(case))


@pytest.mark.parametrize("ctx,n_q,n_kv,hd,bs", [([0], 4, 1, 128, 32), ([513], 32, 8, 128, 128),
                                                ([0, 77, 3000, 255, 256], 32, 8, 128, 64),
                                                ([40] * 70, 7, 1, 64, 32),
                                                ([9000, 1], 16, 16, 64, 128)])
def test_decode_steps(ctx, n_q, n_kv, hd, bs):
    """Without query_start_loc: one row a sequence, the same as with it."""
    print(len(ctx), n_q, n_kv, hd, bs, flush=True)
    c = Case(3, [1] * len(ctx), ctx, n_q, n_kv, hd, bs)
    got = c.run(decode=True)
    c.check(got)
    assert torch.equal(got, c.run())


def test_rows_that_see_nothing_are_zero():
    """seq_lens below the number of query tokens (and 0, and negative)."""
    c = Case(4, [3, 2, 1, 4], [0, 0, 0, 0], 8, 2, 64, 32)
    c.lens = torch.tensor([1, 0, -5, 2], dtype=torch.int32)
    got = c.run()
    c.check(got)
    for row in (0, 1, 3, 4, 5, 6, 7):
        assert not got[row].any()
    assert got[2].any() and got[9].any()


@pytest.mark.parametrize("n,ctx", [([1], [40]), ([6], [90]), ([40], [30]), ([700], [30])])
@pytest.mark.parametrize("hd", [64, 128])
def test_what_is_not_seen_does_not_count(n, ctx, hd):
    """NaN and infinite scales and any codes behind the last token of a page, on pages that no
    sequence lists and at later tokens of other rows' pages."""
    c = Case(5, n + [2], ctx + [3], 16, 4, hd, 32)
    clean = c.run()
    bs = 32
    for r in range(2):
        L = int(c.lens[r])
        for b in range(c.table.shape[1]):
            lo = max(0, min(bs, L - b * bs))
            page = int(c.table[r, b])
            c.scales[:, page, :, lo:] = math.nan if b % 2 else math.inf
            c.codes[:, page, :, lo:] = 0xff
    listed = set(c.table.flatten().tolist())
    for page in range(c.codes.shape[1]):
        if page not in listed:
            c.scales[:, page] = math.nan
    assert torch.equal(clean.view(torch.int16), c.run().view(torch.int16))


@pytest.mark.parametrize("n,n_q,n_kv", [(50, 4, 1), (450, 32, 8)])
def test_later_tokens_do_not_reach_earlier_rows(n, n_q, n_kv):
    """A prompt whose last token's K and V are NaN: only the row that sees it is NaN."""
    c = Case(6, [n], [0], n_q, n_kv, 128, 32)
    assert c.prompts() == (n > 400)
    page, at = int(c.table[0, (n - 1) // 32]), (n - 1) % 32
    for plane in range(2):
        save = c.scales[plane, page, :, at].clone()
        c.scales[plane, page, :, at] = math.nan
        got = c.run().cpu()
        assert got[n - 1].isnan().all()
        assert torch.isfinite(got[:n - 1]).all()
        c.scales[plane, page, :, at] = save


@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("heads,spare", [((8, 2), 1), ((32, 8), 90)])
def test_entries_outside_the_cache(bad, heads, spare):
    """Rows that see a token whose table entry is outside the cache are NaN, the others are
    what they were."""
    c = Case(7, [100, 3], [0, 60], *heads, 128, 32, spare=spare)
    assert c.prompts() == (spare > 1)
    clean = c.run().cpu()
    c.table[0, 2] = bad  # tokens 64..95
    c.table[1, 2:] = bad  # (entries past the length are not looked at)
    c.lens[1] = 64
    got = c.run().cpu()
    assert got[64:100].isnan().all()
    assert torch.equal(got[:64], clean[:64])
    assert torch.isfinite(got[100:]).all()


def test_strided_queries_and_streams():
    """Queries as a slice of the QKV rows; a call on another stream."""
    c = Case(8, [5, 20], [100, 0], 8, 2, 64, 32)
    want = c.run()
    wide = torch.zeros((25, 12, 64), dtype=BF16, device="cuda")
    wide[:, :8] = c.q.cuda()
    ops = _ops()
    cache = ops.Q4KVCache(c.codes.cuda(), c.scales.cuda())
    args = [cache, c.table.cuda(), c.lens.cuda(), c.scale]
    start = c.start.cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.q4_attention(wide[:, :8], *args, query_start_loc=start)
    side.synchronize()
    assert torch.equal(got, want)


def test_capture_with_lengths_that_change():
    """One captured call: lengths from 0 to the capacity, whole and cut, a poisoned
    workspace between the replays."""
    ops = _ops()
    c = Case(9, [1, 1, 1], [6000, 4000, 3], 32, 8, 128, 128)
    q, table, lens = c.q.cuda(), c.table.cuda(), c.lens.cuda()
    cache = ops.Q4KVCache(c.codes.cuda(), c.scales.cuda())
    ws = ops.q4_attention_workspace(q, cache, table)
    assert ws is not None
    out = torch.empty_like(q)
    call = lambda: ops.q4_attention(q, cache, table, lens, c.scale, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for now in ([1, 2, 3], [6001, 4001, 4], [0, 64, 65], [300, 6000, 0], [5, 255, 257]):
        c.lens = torch.tensor(now, dtype=torch.int32)
        lens.copy_(c.lens)
        ws.fill_(255)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        c.check(out, str(now))


def test_a_long_cache():
    """Offsets past 2^31 and 2^32 bytes: pages at both ends of a cache of 5 GB of codes."""
    ops = _ops()
    bs, n_kv, hd = 128, 8, 128
    blocks = 38200
    try:
        codes = torch.zeros((2, blocks, n_kv, bs, hd // 2), dtype=torch.uint8, device="cuda")
        scales = torch.zeros((2, blocks, n_kv, bs, hd // 32), dtype=torch.float16, device="cuda")
    except torch.OutOfMemoryError:
        pytest.skip("needs 6 GB")
    c = Case(10, [1, 1], [300, 200], 32, n_kv, hd, bs)
    used = c.table.flatten().unique().long()
    far = blocks - 1 - torch.arange(used.numel())  # page by page at the end
    far[0] = 0
    codes[:, far.cuda()] = c.codes[:, used].cuda()
    scales[:, far.cuda()] = c.scales[:, used].cuda()
    new = torch.zeros(c.codes.shape[1], dtype=torch.int64)
    new[used] = far
    cache = ops.Q4KVCache(codes, scales)
    got = ops.q4_attention(c.q.cuda(), cache, new[c.table.long()].to(torch.int32).cuda(),
                           c.lens.cuda(), c.scale)
    assert torch.equal(got, c.run(decode=True))
    # a write and a read of the last slot
    key = torch.randn((1, n_kv, hd), device="cuda").to(BF16)
    slot = torch.tensor([blocks * bs - 1], device="cuda")
    ops.reshape_and_cache_q4(key, key, cache, slot)
    small = ops.q4_kv_cache(1, bs, n_kv, hd, "cuda")
    ops.reshape_and_cache_q4(key, key, small, slot * 0)
    for a, b in zip(ops.q4_kv_read(cache, slot), ops.q4_kv_read(small, slot * 0)):
        assert torch.equal(a, b)


def test_refusals():
    ops = _ops()
    c = Case(11, [1, 1], [5, 9], 8, 2, 64, 32)
    q, table, lens, start = c.q.cuda(), c.table.cuda(), c.lens.cuda(), c.start.cuda()
    cache = ops.Q4KVCache(c.codes.cuda(), c.scales.cuda())
    f = lambda **k: ops.q4_attention(*({**dict(q=q, cache=cache, block_table=table, seq_lens=lens,  # noqa: E731
                                               scale=0.1), **k}.values()))
    f()
    bad = [dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(q=q[:, :, :32]),
           dict(q=q.transpose(0, 1)), dict(cache=None), dict(cache=(cache.codes, cache.scales)),
           dict(block_table=table.long()), dict(block_table=table[0]),
           dict(block_table=table.cpu()), dict(seq_lens=lens[:1]), dict(seq_lens=lens.long()),
           dict(q=q[:1]), dict(s=start[:2]), dict(s=start.long()), dict(s=start, w=torch.empty(4)),
           dict(s=start, w=None, out=torch.empty_like(q)[:1])]
    for i, change in enumerate(bad):
        with pytest.raises(ValueError):
            f(**change)
            print("not refused:", i)
    for change in (dict(scale=0.0), dict(scale=math.nan), dict(q=q[:, :7].contiguous())):
        with pytest.raises(pkg("native").SmxError):
            f(**change)


@pytest.mark.parametrize("n,ctx,n_q,n_kv,hd,bs", [
    (50, 0, 4, 1, 128, 32), (450, 0, 32, 8, 128, 32), (1500, 0, 16, 4, 64, 64),
    (300, 3000, 32, 8, 128, 64), (2100, 0, 32, 8, 128, 128), (2100, 0, 32, 8, 64, 32)])
def test_blocks_of_v_without_a_value(n, ctx, n_q, n_kv, hd, bs):
    """A NaN scale of V is one block's of 32 dims: the rows that see its token are NaN there,
    and everything else is what it was."""
    c = Case(8, [n], [ctx], n_q, n_kv, hd, bs)
    assert c.prompts() == (n > 50)
    clean = c.run().cpu()
    for t, block in ((n + ctx - 2, 0), (ctx + n // 2, hd // 32 - 1), (ctx + 5, 1)):
        where = (1, int(c.table[0, t // bs]), n_kv - 1, t % bs, block)
        save = c.scales[where].clone()
        c.scales[where] = math.nan
        got = c.run().cpu()
        c.scales[where] = save
        heads, dims = slice(n_q - n_q // n_kv, n_q), slice(32 * block, 32 * block + 32)
        assert got[t - ctx:, heads, dims].isnan().all()
        got[t - ctx:, heads, dims] = clean[t - ctx:, heads, dims]
        assert torch.isfinite(got).all()
        # (the weights of a tile are rescaled or not by rows that are NaN now: one rounding)
        torch.testing.assert_close(got, clean, rtol=2.0 ** -7, atol=2.0 ** -9)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("most", [900, 3000])
def test_wide_tables(hd, most):
    """Tables much wider than their sequences are long (a model's full width): calls are cut
    into more parts, most of which have nothing."""
    n = [1] * 19 + [3, 0]
    ctx = [0, 31, 32, 127, 128, 129, 255, 500] + [most - 83 * i % most for i in range(13)]
    c = Case(12, n, ctx, 8, 4, hd, 32)
    narrow = c.run()
    wide = torch.full((len(n), 500 - c.table.shape[1]), -1, dtype=torch.int32)
    c.table = torch.cat((c.table, wide), 1)
    got = c.run()
    c.check(got)
    c.check(narrow)
