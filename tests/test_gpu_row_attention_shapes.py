"""The row attentions' workgroups of 128 rows, which serve most prompts and large
batches under a prefix: heads of 64 and 128 with pages of 32 (a 64-token tile of two
pages) and of 128, whole tiles and cut ones.  Sizes that take them: sequences of 65
to 128 rows in 256 workgroups of 64, fresh prompts above 800 of those, prompts behind
a context above 512, one prompt of over 1024 rows before 8192 tokens; prefixes of 1.5
million (row, token) pairs."""
import math

import pytest
import torch

from _rows import assert_rows, gather
from _util import pkg
from test_gpu_prompt_attention import _case, _run
from test_gpu_shared_prefix import _case as _prefix_case
from test_gpu_shared_prefix import _run as _prefix_run

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
SHAPES = [(128, 128), (128, 32), (64, 128), (64, 32)]  # head_dim, block_size


def _ops():
    return pkg("native.torch_ops")


def _attend64(q, k, v, scale, seen):
    """_rows.attend64 without a copy of K and V for every q head."""
    n_kv, hd = k.shape[1:]
    q = q.double().view(q.shape[0], n_kv, -1, hd)
    s = torch.einsum("rngd,tnd->ngrt", q, k) * scale
    s = torch.where(seen, s, -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot > 0, tot, 1.0)
    return tuple(torch.einsum("ngrt,tnd->rngd", p, x).reshape(q.shape[0], -1, hd)
                 for x in (v, v.abs()))


def _prompt64(q, k, v, table, start, lens, scale):
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for r, L in enumerate(lens.tolist()):
        a, b = int(start[r]), int(start[r + 1])
        if L <= 0 or b <= a:
            continue
        seen = torch.arange(L)[None] <= torch.arange(L - (b - a), L)[:, None]
        out[a:b], mag[a:b] = _attend64(q[a:b], gather(k, table[r], L), gather(v, table[r], L),
                                       scale, seen)
    return out, mag


def _prefix64(q, k, v, ptable, plen, table, lens, scale):
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    P, bs = int(plen), k.shape[1]
    pk, pv = gather(k, ptable, P), gather(v, ptable, P)
    for r, L in enumerate(lens.tolist()):
        if L <= 0:
            continue
        t = torch.arange(min(P, L), L)
        page = table[r][t // bs].long()
        kk, vv = (torch.cat((pre[:L], c[page, t % bs].double())) for pre, c in ((pk, k), (pv, v)))
        out[r:r + 1], mag[r:r + 1] = _attend64(q[r:r + 1], kk, vv, scale,
                                               torch.ones((1, L), dtype=torch.bool))
    return out, mag


PROMPTS = [
    # n, ctx, n_q, n_kv: 65 to 128 rows a sequence, whole tiles
    ([40, 33, 50, 37], [0, 5, 70, 200], 64, 32),
    # the same, cut for the long one (14 parts)
    ([40, 33, 50, 37], [10, 3500, 64, 900], 64, 32),
    # fresh prompts, a group of 3
    ([300, 1, 0, 560], [0, 0, 0, 0], 96, 32),
    # behind a context, a group of 5
    ([100, 120], [400, 650], 160, 32),
    # one long range, cut (16 parts), a group of 7
    ([300], [8000], 14, 2),
]


@pytest.mark.parametrize("hd,bs", SHAPES)
@pytest.mark.parametrize("case", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
def test_prompts(case, hd, bs):
    print(f"prompts {case} {hd} {bs}", flush=True)
    c = _case(21, *case, hd, bs, pad=3)
    out = torch.full(c[0].shape, 7.0, dtype=BF16, device="cuda")
    got = _run(*c, 0.1, out=out).cpu()
    total = sum(case[0])
    assert (got[total:] == 7).all()
    ref, mag = _prompt64(*c, 0.1)
    assert_rows(got[:total], ref[:total], mag[:total], f"{case} {hd} {bs}")


WHOLE, CUT = [0, 5, 70, 200], [10, 3500, 64, 900]


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("ctx,hd,bs", [(WHOLE, *x) for x in SHAPES]
                         + [(CUT, 128, 128), (CUT, 64, 32)])
def test_prompts_unseen_values(ctx, bad, hd, bs):
    """Infinities and NaN in slots behind a sequence's end and in its last but one
    token, which only its last two rows see."""
    print(f"unseen {ctx} {bad} {hd} {bs}", flush=True)
    q, k, v, table, start, lens = _case(22, [40, 33, 50, 37], ctx, 64, 32, hd, bs)
    ref, mag = _prompt64(q, k, v, table, start, lens, 0.1)
    tail = []
    for r, L in enumerate(lens.tolist()):
        for t in range(L, min(table.shape[1] * bs, L + 200)):
            k[table[r, t // bs], t % bs] = bad
            v[table[r, t // bs], t % bs] = bad
        k[table[r, (L - 2) // bs], (L - 2) % bs, :, 3] = bad
        v[table[r, (L - 2) // bs], (L - 2) % bs, :, 5] = bad
        tail += [int(start[r + 1]) - 2, int(start[r + 1]) - 1]
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    keep = [i for i in range(q.shape[0]) if i not in tail]
    assert_rows(got[keep], ref[keep], mag[keep], f"{bad}")
    if math.isnan(bad):
        assert torch.isnan(got[tail]).all()


@pytest.mark.parametrize("hd,bs", SHAPES)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_prompts_seen_values(bad, hd, bs):
    """An infinite (NaN) V of a token: in its dim of the rows that see it."""
    q, k, v, table, start, lens = _case(23, [40, 33, 50, 37], [0, 5, 70, 200], 64, 32, hd, bs)
    ref, mag = _prompt64(q, k, v, table, start, lens, 0.1)
    v[table[2, 90 // bs], 90 % bs, :, 9] = bad  # seen by rows 20 .. 49 of sequence 2
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    first, end = int(start[2]) + 20, int(start[3])
    hit = got[first:end, :, 9].float()
    assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
    got[first:end, :, 9] = ref[first:end, :, 9].to(BF16)
    assert_rows(got, ref, mag, "others")


@pytest.mark.parametrize("ctx,hd,bs", [(WHOLE, *x) for x in SHAPES]
                         + [(CUT, 128, 32), (CUT, 64, 128)])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_prompts_bad_pages(entry, ctx, hd, bs):
    """One bad page, the first or the second of a tile's two: NaN from its first token
    on, the rows before it as they are."""
    print(f"bad pages {entry} {ctx} {hd} {bs}", flush=True)
    q, k, v, table, start, lens = _case(24, [40, 33, 50, 37], ctx, 64, 32, hd, bs)
    ref, mag = _prompt64(q, k, v, table, start, lens, 0.1)
    keep = []
    for r, n in enumerate([40, 33, 50, 37]):
        page = [0, (ctx[1] + 20) // bs, (ctx[2] + 30) // bs, ctx[3] // bs][r]
        if r == 0:
            page = 10 ** 9  # none
        else:
            table[r, page] = entry
        keep += [int(start[r]) + i for i in range(n) if ctx[r] + i < page * bs]
        table[r, int(lens[r] - 1) // bs + 1:] = entry  # past the end
    got = _run(q, k, v, table, start, lens, 0.1).cpu()
    lost = [i for i in range(q.shape[0]) if i not in keep]
    assert torch.isnan(got[lost]).all() and len(lost) > 40
    assert_rows(got[keep], ref[keep], mag[keep], f"entry {entry}")


@pytest.mark.parametrize("hd,bs", SHAPES)
def test_prompts_short_lengths_and_strides(hd, bs):
    """Lengths below the number of query tokens, and q as a slice of wider rows."""
    q, k, v, table, start, lens = _case(25, [40, 33, 50, 37], [0, 5, 70, 200], 64, 32, hd, bs)
    lens[0], lens[1], lens[3] = 33, 0, -5
    wide = torch.zeros((q.shape[0], 80 * hd), dtype=BF16, device="cuda")
    view = wide[:, 8 * hd:72 * hd].view(q.shape)
    view.copy_(q)
    got = _ops().prompt_attention(view, *[x.cuda() for x in (k, v, table, start, lens)], 0.1).cpu()
    ref, mag = _prompt64(q, k, v, table, start, lens, 0.1)
    for a, b in ((0, 7), (40, 73), (123, 160)):
        assert torch.equal(got[a:b], torch.zeros_like(got[a:b]))
    assert_rows(got, ref, mag, "short lengths")


@pytest.mark.parametrize("hd,bs", [(128, 128), (64, 32)])
@pytest.mark.parametrize("case", [PROMPTS[1], PROMPTS[2], PROMPTS[4]], ids=["cut", "fresh", "long"])
def test_prompts_captured(case, hd, bs):
    """A captured call, replayed on other lengths, offsets and rows with eager calls
    between: the eager bits each time."""
    q, k, v, table, start, lens = [x.cuda() for x in _case(26, *case, hd, bs)]
    ops = _ops()
    ws = ops.prompt_attention_workspace(q, k, table)
    if ws is not None:
        ws.fill_(255)
    out = torch.empty_like(q)
    call = lambda: ops.prompt_attention(q, k, v, table, start, lens, 0.1, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        lens.sub_(13 * i)
        if i == 2 and start.numel() > 2:
            start[1] -= 5
        q.mul_(-1)
        ref = ops.prompt_attention(q, k, v, table, start, lens, 0.1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), ref.view(torch.int16)), f"replay {i}"


PREFIXES = [
    # prefix, suffix lengths, n_q, n_kv: 384 rows, parts of one or two rounds
    (3950, [(37 * i) % 90 for i in range(48)], 16, 2),
    # 128 rows, parts of three rounds
    (11800, [(29 * i) % 150 for i in range(16)], 32, 4),
    # 800 rows, more sequences than one round of the search
    (2000, [(5 * i) % 70 for i in range(100)], 8, 1),
]


def _prefix_check(case, what):
    ref, mag = _prefix64(*case, 0.1)
    assert_rows(_prefix_run(case), ref, mag, what)


@pytest.mark.parametrize("hd,bs", SHAPES)
@pytest.mark.parametrize("case", PREFIXES, ids=[str(i) for i in range(len(PREFIXES))])
def test_prefixes(case, hd, bs):
    print(f"prefix {case[0]} {hd} {bs}", flush=True)
    _prefix_check(_prefix_case(31, *case, hd, bs, own_prefix_entries=False), f"{hd} {bs}")


@pytest.mark.parametrize("hd,bs", SHAPES)
def test_prefixes_lengths_below_the_prefix(hd, bs):
    case = _prefix_case(32, *PREFIXES[0], hd, bs)
    lens = case[6]
    lens[0], lens[1], lens[2], lens[5], lens[9] = 77, 0, -3, 3949, 1
    lens[20:40] = torch.arange(20, dtype=torch.int32) * 200
    _prefix_check(case, "short rows")


@pytest.mark.parametrize("hd,bs", SHAPES)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_prefixes_unseen_values(bad, hd, bs):
    """Behind the prefix's end in its last page, in the own pages' slots below it, and
    behind every sequence's end."""
    case = _prefix_case(33, *PREFIXES[0], hd, bs)
    q, k, v, ptable, plen, table, lens = case
    ref, mag = _prefix64(*case, 0.1)
    at = 3950 % bs
    for c in (k, v):
        c[ptable[-1], at:] = bad
        for r in range(48):
            c[table[r, 3950 // bs], :at] = bad
            for t in range(int(lens[r]), table.shape[1] * bs):
                c[table[r, t // bs], t % bs] = bad
    assert_rows(_prefix_run(case), ref, mag, f"{bad}")


@pytest.mark.parametrize("hd,bs", SHAPES)
def test_prefixes_seen_values_and_bad_pages(hd, bs):
    """An infinite V of the prefix reaches the rows longer than its token, a bad
    page of a sequence that sequence alone, one of the prefix whoever sees it."""
    case = _prefix_case(34, *PREFIXES[0], hd, bs, own_prefix_entries=False)
    q, k, v, ptable, plen, table, lens = case
    lens[4], lens[5] = 3000, 3001
    ref, mag = _prefix64(*case, 0.1)
    v[ptable[3000 // bs], 3000 % bs, 1, 7] = math.inf
    table[11, 3950 // bs] = 10 ** 6  # 47 own tokens
    got = _prefix_run(case).cpu()
    assert torch.isnan(got[11]).all()
    hit = [r for r in range(48) if r not in (4, 11)]
    dim = got[..., 7]
    assert (dim[hit][:, 8:].float() == math.inf).all()
    got[..., 7] = torch.where(dim == math.inf, ref[..., 7].to(BF16), dim)
    rest = [r for r in range(48) if r != 11]
    assert_rows(got[rest], ref[rest], mag[rest], "others")
    ptable[2 if bs == 128 else 8] = -1  # tokens 256 on
    lens[7] = 256
    got = _prefix_run(case).cpu()
    assert torch.isfinite(got[7]).all()
    assert torch.isnan(got[[r for r in range(48) if r != 7]]).all()


@pytest.mark.parametrize("hd,bs", [(128, 128), (64, 128), (128, 32)])
def test_prefixes_captured(hd, bs):
    case = [x.cuda() for x in _prefix_case(35, *PREFIXES[0], hd, bs)]
    ops = _ops()
    ws = ops.shared_prefix_attention_workspace(case[0], case[1], case[3], case[5])
    ws.fill_(255)
    out = torch.empty_like(case[0])
    call = lambda: ops.shared_prefix_attention(*case, 0.1, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        case[4].sub_(500 * i)  # a shorter prefix: the rest is read from the own pages
        case[6].sub_(40 * i)
        case[0].mul_(-1)
        ref = ops.shared_prefix_attention(*case, 0.1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), ref.view(torch.int16)), f"replay {i}"
        want, mag = _prefix64(*[x.cpu() for x in case], 0.1)
        assert_rows(out, want, mag, f"replay {i}")
