"""What a server needs to hold more sequences and more hypotheses a sequence in the
same memory, as cases that can be timed and checked:

  attend   attention of packed query rows (decode steps, drafts, chunks) over a paged
           cache held in 4 bits
  write    keys and values into that cache, and the tokens' values read back
  beams    a beam search's selection over beams and vocabulary
  fork     block tables of the chosen beams: pages shared, tails copied, dead ones freed
  compact  the pages in use moved to the front of the pool

  listed()             the cases, dicts of plain values
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  inputs on the GPU, from the seed
  run(state)           one pass: the plain form, or with `own` the framework's calls
  work(case)           bytes and flops that the pass cannot do without
  exact(case, seed)    the outputs in 64 bits, written apart from the plain form

Shapes are the 4B decoder's (32 q / 8 kv heads of 128, pages of 128 tokens,
vocabulary 151936, contexts to 32768) and generic ones.

The 4-bit cache: blocks of 32 channels of one head of a token share an fp16 scale d and
hold codes c of 0..15 that stand for d * (c - 8).  d is fp16(m / -8), m the block's
first value of largest magnitude, and c = floor(x / d + 8.5) kept within 0..15.
codes uint8 [2, pages, n_kv, page, hd / 2], scales fp16 [2, pages, n_kv, page, hd / 32],
K first.  V's codes are in channel order, the lower half of a byte first.  K's dword
g * (hd / 32) + b holds channels 32 b + 8 g .. + 7, the even ones in its lower half.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
INF = math.inf


# --------------------------------------------------------------------- cases
def _attend_case(name, seqs, lo, hi, ctx_lo, ctx_hi, n_q=32, n_kv=8, hd=128, bs=128, pad=0):
    return dict(name=name, kind="attend", seqs=seqs, lo=lo, hi=hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
                n_q=n_q, n_kv=n_kv, hd=hd, bs=bs, pad=pad)


def _write_case(name, tokens, pad, n_kv=8, hd=128, bs=128):
    return dict(name=name, kind="write", tokens=tokens, pad=pad, n_kv=n_kv, hd=hd, bs=bs)


def _beams_case(name, seqs, beams, width, vocab, wide=False, banned=0.0, done=0.0):
    return dict(name=name, kind="beams", seqs=seqs, beams=beams, width=width, vocab=vocab,
                wide=wide, banned=banned, done=done)


def _fork_case(name, seqs, beams, lo, hi, layers, n_kv=8, hd=128, bs=128):
    return dict(name=name, kind="fork", seqs=seqs, beams=beams, lo=lo, hi=hi, layers=layers,
                n_kv=n_kv, hd=hd, bs=bs)


def _compact_case(name, seqs, lo, hi, spare, layers, n_kv=8, hd=128, bs=128):
    return dict(name=name, kind="compact", seqs=seqs, lo=lo, hi=hi, spare=spare, layers=layers,
                n_kv=n_kv, hd=hd, bs=bs)


def listed() -> list[dict]:
    return [
        # one session's decode step behind a short context: the smallest, latency
        _attend_case("attend_1seq", 1, 1, 1, 512, 512),
        # a large batch's decode step behind long contexts
        _attend_case("attend_48seq", 48, 1, 1, 2000, 32000),
        # one chunk of a long prompt, behind what earlier chunks left in the cache
        _attend_case("attend_chunk", 1, 509, 509, 16000, 16000),
        # another layout, ragged: single tokens, drafts and prompts in one padded pass
        _attend_case("attend_hd64", 7, 1, 700, 0, 900, n_q=14, n_kv=2, hd=64, bs=32, pad=5),
        # a decode step's tokens
        _write_case("write_16", 16, 0),
        # a prefill pass, padded
        _write_case("write_8k", 8000, 192),
        # one session's beam search, candidates for beams that end
        _beams_case("beams_4", 1, 4, 8, 151936),
        # a batch's: some tokens are not allowed, some beams have ended
        _beams_case("beams_512", 64, 8, 16, 151936, banned=0.2, done=0.1),
        # one session's beams, all of the model's layers
        _fork_case("fork_4", 1, 4, 700, 700, 36),
        # a batch's; few layers, so that a state fits the card three times
        _fork_case("fork_512", 64, 8, 100, 4000, 2),
        # a small pool after requests have come and gone
        _compact_case("compact_16", 16, 1, 900, 40, 4),
        # a large pool, half of it free
        _compact_case("compact_256", 256, 1, 2000, 1500, 2),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8, 128), (32, 8, 128), (32, 8, 128), (16, 16, 128), (14, 2, 64), (24, 8, 64),
          (40, 8, 128), (8, 1, 128), (16, 4, 64)]


def draw(rng) -> dict:
    kind = rng.choice(["attend", "attend", "attend", "write", "beams", "beams", "fork", "compact"])
    n_q, n_kv, hd = rng.choice(_HEADS)
    bs = rng.choice([32, 64, 128, 128, 256])
    if kind in ("fork", "compact"):
        bs = min(bs, 131072 // (n_kv * hd))
    if kind == "attend":
        seqs = _log_int(rng, 1, 64)
        hi = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 1, max(1, 2048 // seqs))])
        lo = rng.choice([1, hi])
        # the plain form pads: rows and tokens of the longest, of every sequence
        most = min(32000, 1_500_000 // seqs, 260_000_000 // (seqs * hi * n_q)) - hi
        ctx = rng.choice([0, _log_int(rng, 1, most), _log_int(rng, 1, most)]) if most > 1 else 0
        c = _attend_case("", seqs, lo, hi, ctx // rng.choice([1, 3, 20]), ctx, n_q, n_kv, hd, bs,
                         rng.choice([0, 0, 3, 64]))
    elif kind == "write":
        c = _write_case("", _log_int(rng, 1, 8192), rng.choice([0, 0, 7, 100]), n_kv, hd, bs)
    elif kind == "beams":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
        wide = rng.random() < 0.3
        vocab = _log_int(rng, 300, 152000)
        seqs = _log_int(rng, 1, max(1, min(64, 70_000_000 // (beams * vocab * (1 + wide)))))
        c = _beams_case("", seqs, beams, rng.choice([beams, 2 * beams, min(64, 3 * beams + 1)]),
                        vocab, wide, rng.choice([0.0, 0.0, 0.2, 0.999]), rng.choice([0.0, 0.2]))
    elif kind == "fork":
        beams = rng.choice([1, 2, 4, 5, 8])
        hi = _log_int(rng, 1, 4000)
        c = _fork_case("", _log_int(rng, 1, min(48, 200_000 // (beams * hi))), beams,
                       rng.choice([1, hi, max(1, hi // 9)]), hi, rng.randint(1, 2), n_kv, hd, bs)
    else:
        hi = _log_int(rng, 1, 2000)
        c = _compact_case("", _log_int(rng, 1, min(200, 100_000 // hi)), rng.choice([1, hi]), hi,
                          _log_int(rng, 1, 150_000 // bs), rng.randint(1, 2), n_kv, hd, bs)
    del c["name"]
    return c


# -------------------------------------------------------------------- inputs
def _gen(seed: int, salt: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) & 0x7FFFFFFF) * 1000003 + salt)
    return g


def _spread(n: int, lo: int, hi: int, salt: int) -> list[int]:
    """n lengths from lo to hi, both among them where n allows, spread over their
    logarithm; the same for every seed, so that a case is one amount of work."""
    r = random.Random(1000003 * n + 8191 * lo + 31 * hi + salt)
    out = [hi] + [min(hi, max(lo, _log_int(r, max(lo, 1), max(hi, 1)))) for _ in range(n - 2)]
    out += [lo] if n > 1 else []
    r.shuffle(out)
    return out


def _i32(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _normal(shape, seed, salt, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0,
                                                                  generator=_gen(seed, salt))


def _codes(x):
    """(codes 0..15, fp16 scales) of x [..., hd], blocks of 32."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().argmax(-1, keepdim=True)
    d = (b.gather(-1, top) / -8).clamp(-65504, 65504).half()
    df = d.float()
    c = torch.where(df == 0, 8.0, torch.floor(b / torch.where(df == 0, 1.0, df) + 8.5))
    return c.clamp(0, 15).to(torch.uint8).flatten(-2), d.squeeze(-1)


def _k_order(hd: int) -> torch.Tensor:
    """The channel of each of a K row's hd half-bytes."""
    at = torch.arange(hd, device="cuda")
    dword, nib = at // 8, at % 8
    g, b = dword // (hd // 32), dword % (hd // 32)
    return 32 * b + 8 * g + torch.where(nib < 4, 2 * nib, 2 * (nib - 4) + 1)


def _pack(c, is_key):
    if is_key:
        c = c[..., _k_order(c.shape[-1])]
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _unpack(p, is_key):
    c = torch.stack((p & 15, p >> 4), -1).flatten(-2)
    if not is_key:
        return c
    out = torch.empty_like(c)
    out[..., _k_order(c.shape[-1])] = c
    return out


def _rows_of(cache_part, page, at):
    """Rows [..., n_kv, width] of a [pages, n_kv, bs, width] tensor."""
    return cache_part.transpose(1, 2)[page, at]


def _values(codes, scales, is_key):
    c = _unpack(codes, is_key).float() - 8
    return (c.unflatten(-1, (-1, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _ops():
    import importlib
    import os

    os.environ.setdefault("SMX_ALLOW_UNVALIDATED", "1")  # the library as built is what is measured
    import __graft_entry__

    return importlib.import_module(__graft_entry__.load_package().__name__ + ".native.torch_ops")


def prepare(case: dict, seed: int) -> dict:
    s = _PREPARE[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    if own:
        s["ops"] = ops = _ops()
        if case["kind"] in ("attend", "write"):
            s["cache"] = ops.Q4KVCache(s["codes"], s["scales"])
        if case["kind"] == "attend":
            s["workspace"] = ops.q4_attention_workspace(s["q"], s["cache"], s["table"], s["start"])
        elif case["kind"] == "beams":
            s["workspace"] = ops.beam_select_workspace(s["logits"], s["beams"], s["width"])
        elif case["kind"] in ("fork", "compact"):
            s["set"] = ops.PageSet(list(s["caches"].unbind(0)), page_dim=1)
    return s


def _prep_attend(case, seed):
    n = _spread(case["seqs"], case["lo"], case["hi"], 1)
    ctx = _spread(case["seqs"], case["ctx_lo"], case["ctx_hi"], 2)
    lens = [a + b for a, b in zip(n, ctx)]
    bs, hd, n_kv = case["bs"], case["hd"], case["n_kv"]
    held = [-(-x // bs) for x in lens]
    width = max(held) + 1
    blocks = sum(held) + 3
    codes = torch.empty((2, blocks, n_kv, bs, hd // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((2, blocks, n_kv, bs, hd // 32), dtype=torch.float16, device="cuda")
    for i in range(2):
        c, scales[i] = _codes(_normal((blocks, n_kv, bs, hd), seed, 10 + i))
        codes[i] = _pack(c, i == 0)
    perm = torch.randperm(blocks, generator=_gen(seed, 2), device="cuda").to(torch.int32)
    h = _i32(held)[:, None]
    col = torch.arange(width, device="cuda")[None]
    first = torch.cumsum(h, 0) - h
    table = torch.where(col < h, perm[(first + col).clamp(max=blocks - 1)], -1).to(torch.int32)
    start = [0]
    for x in n:
        start.append(start[-1] + x)
    rows = sum(n) + case["pad"]
    # a decode batch needs no offsets: a row a sequence
    decode = case["hi"] == 1 and case["pad"] == 0
    return dict(q=_normal((rows, case["n_q"], hd), seed, 3), codes=codes, scales=scales,
                table=table.contiguous(), start=None if decode else _i32(start), lens=_i32(lens),
                n=_i32(n), most=max(n), longest=max(lens), scale=1.0 / math.sqrt(hd),
                out=torch.zeros((rows, case["n_q"], hd), dtype=BF16, device="cuda"))


def _prep_write(case, seed):
    t, n_kv, hd, bs = case["tokens"], case["n_kv"], case["hd"], case["bs"]
    blocks = -(-t // bs) + 4
    slots = torch.randperm(blocks * bs, generator=_gen(seed, 2), device="cuda")[:t]
    # channels of unlike sizes, as keys have them
    size = torch.exp(_normal((n_kv, hd), seed, 5, torch.float32))
    kv = [(_normal((t + case["pad"], n_kv, hd), seed, 3 + i, torch.float32) * (size if i == 0 else
           0.3)).to(BF16) for i in range(2)]
    none = torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")
    return dict(key=kv[0], value=kv[1], slots=torch.cat((slots, none)),
                codes=torch.zeros((2, blocks, n_kv, bs, hd // 2), dtype=torch.uint8, device="cuda"),
                scales=torch.zeros((2, blocks, n_kv, bs, hd // 32), dtype=torch.float16,
                                   device="cuda"))


def _prep_beams(case, seed):
    rows, vocab = case["seqs"] * case["beams"], case["vocab"]
    g = _gen(seed, 1)
    x = torch.empty((rows, vocab), dtype=torch.float32, device="cuda").normal_(0.0, 3.0,
                                                                             generator=g)
    if case["banned"]:  # constrained decoding: most often the same tokens for all
        x.masked_fill_(torch.rand((1, vocab), generator=g, device="cuda") < case["banned"], -INF)
    scores = -20.0 * torch.rand(rows, generator=g, device="cuda")
    done = None
    if case["done"]:
        done = torch.rand(rows, generator=g, device="cuda") < case["done"]
        # and beams that do not live yet: a step after the first with few candidates
        dead = torch.rand(rows, generator=g, device="cuda") < case["done"] / 4
        scores = torch.where(dead, -INF, scores)
    return dict(logits=x if case["wide"] else x.to(BF16), scores=scores, done=done,
                beams=case["beams"], width=case["width"], pad_id=1)


def _fork_lens(case):
    return [x for x in _spread(case["seqs"], case["lo"], case["hi"], 1)
            for _ in range(case["beams"])]


def _parents(case, seed):
    """Each beam of the next step's parent: some twice and more, some never."""
    r = random.Random(97 * seed + 5)
    out = []
    for i in range(case["seqs"]):
        out += [i * case["beams"] + min(r.randrange(case["beams"]), r.randrange(case["beams"]))
                for _ in range(case["beams"])]
    return out


def _caches(case, seed, blocks):
    shape = (case["layers"], 2, blocks, case["bs"], case["n_kv"], case["hd"])
    return _normal(shape, seed, 4)


def _prep_fork(case, seed):
    lens, beams, bs = _fork_lens(case), case["beams"], case["bs"]
    held = [-(-x // bs) for x in lens]
    width = max(held) + 2
    # a sequence's beams share their pages up to some earlier fork, the rest are their own
    r = random.Random(31 * len(lens) + max(lens))
    table, used = [], 0
    for i in range(case["seqs"]):
        h = held[i * beams]
        common = r.randint(h // 2, h - 1) if h > 1 else 0
        shared = list(range(used, used + common))
        used += common
        for _ in range(beams):
            mine = list(range(used, used + h - common))
            used += h - common
            table.append(shared + mine + [-1] * (width - h))
    rows = len(lens)
    blocks = used + rows + 5
    perm = torch.randperm(blocks, generator=_gen(seed, 2), device="cuda").to(torch.int32)
    table = _i32(table)
    table = torch.where(table < 0, -1, perm[table.clamp(min=0)]).to(torch.int32)
    free = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
    free[:blocks - used] = perm[used:]
    return dict(parents=_i32(_parents(case, seed)), lens=_i32(lens), num_pages=_i32(held),
                free_pages=free, free_count=_i32([blocks - used]), table=table, blocks=blocks,
                bs=bs, caches=_caches(case, seed, blocks))


def _prep_compact(case, seed):
    lens = _spread(case["seqs"], case["lo"], case["hi"], 1)
    held = [-(-x // case["bs"]) for x in lens]
    width, used = max(held) + 1, sum(held)
    blocks = used + case["spare"]
    perm = torch.randperm(blocks, generator=_gen(seed, 2), device="cuda").to(torch.int32)
    h = _i32(held)[:, None]
    col = torch.arange(width, device="cuda")[None]
    first = torch.cumsum(h, 0) - h
    table = torch.where(col < h, perm[(first + col).clamp(max=blocks - 1)], -1).to(torch.int32)
    return dict(num_pages=_i32(held), table=table.contiguous(), blocks=blocks,
                caches=_caches(case, seed, blocks))


_PREPARE = {"attend": _prep_attend, "write": _prep_write, "beams": _prep_beams,
            "fork": _prep_fork, "compact": _prep_compact}


# ---------------------------------------------------------------------- run
def run(state: dict):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_attend(s):
    return s["ops"].q4_attention(s["q"], s["cache"], s["table"], s["lens"], s["scale"],
                                 query_start_loc=s["start"], workspace=s["workspace"],
                                 out=s["out"])


def _own_write(s):
    s["ops"].reshape_and_cache_q4(s["key"], s["value"], s["cache"], s["slots"])
    return s["ops"].q4_kv_read(s["cache"], s["slots"])


def _own_beams(s):
    r = s["ops"].beam_select(s["logits"], s["scores"], s["beams"], s["width"], done=s["done"],
                             pad_id=s["pad_id"], workspace=s["workspace"])
    return [r.parents, r.tokens, r.scores]


def _own_fork(s):
    r = s["ops"].fork_pages(s["parents"], s["lens"], s["num_pages"], s["free_pages"],
                            s["free_count"], s["table"], s["blocks"], s["bs"])
    s["ops"].copy_pages(s["set"], r.copies)
    return [r.block_table, r.num_pages, r.lens, r.free_pages, r.free_count, r.copies, s["caches"]]


def _own_compact(s):
    r = s["ops"].compact_pages(s["num_pages"], s["table"], s["blocks"])
    s["ops"].copy_pages(s["set"], r.moves)
    return [r.block_table, r.free_pages, r.free_count, r.moves, s["caches"]]


def _plain_attend(s):
    bs, scale = s["codes"].shape[3], s["scale"]
    rows, n_q, hd = s["q"].shape
    n_kv = s["codes"].shape[2]
    n, lens, most, longest = s["n"].long(), s["lens"].long(), s["most"], s["longest"]
    seqs = n.numel()
    pos = torch.arange(longest, device="cuda")
    page = s["table"][:, pos // bs].clamp(min=0).long()  # [seqs, longest]
    k, v = (_values(_rows_of(s["codes"][i], page, (pos % bs).expand_as(page)),
                    _rows_of(s["scales"][i], page, (pos % bs).expand_as(page)), i == 0)
            .transpose(1, 2).contiguous() for i in range(2))  # [seqs, n_kv, longest, hd]
    first = torch.cumsum(n, 0) - n
    at = torch.arange(most, device="cuda")
    row = torch.where(at < n[:, None], first[:, None] + at, rows)  # [seqs, most]
    q = torch.cat((s["q"].float(), torch.zeros_like(s["q"][:1], dtype=torch.float32)))[row]
    q = q.view(seqs, most, n_kv, -1, hd).permute(0, 2, 1, 3, 4).reshape(seqs, n_kv, -1, hd)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    seen = pos < (lens - n)[:, None, None] + at[:, None] + 1  # [seqs, most, longest]
    x = x.view(seqs, n_kv, most, -1, longest).masked_fill_(~seen[:, None, :, None], -INF)
    x = x.sub_(x.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(seqs, n_kv, -1, longest), v).view(seqs, n_kv, most, -1, hd)
    o = (o / torch.where(total > 0, total, 1.0)).permute(0, 2, 1, 3, 4).reshape(seqs, most, n_q, hd)
    out = torch.zeros((rows + 1, n_q, hd), dtype=BF16, device="cuda")
    out[row] = o.to(BF16)
    out[rows] = 0
    return out[:rows]


def _plain_write(s):
    ok = s["slots"] >= 0
    slots = torch.where(ok, s["slots"], 0)
    bs = s["codes"].shape[3]
    page, at = slots[ok] // bs, slots[ok] % bs
    for i, x in enumerate((s["key"], s["value"])):
        c, d = _codes(x[ok])
        s["codes"][i].transpose(1, 2)[page, at] = _pack(c, i == 0)
        s["scales"][i].transpose(1, 2)[page, at] = d
    return [torch.where(ok[:, None, None], _values(
        _rows_of(s["codes"][i], slots // bs, slots % bs),
        _rows_of(s["scales"][i], slots // bs, slots % bs), i == 0), 0.0) for i in range(2)]


def _order(x):
    """Integers in the order of x's values, -0 as 0."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    return torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)


def _plain_beams(s):
    x, beams, width = s["logits"], s["beams"], s["width"]
    rows, vocab = x.shape
    top = x.amax(-1, keepdim=True).double()
    lse = torch.log((x - top).exp_().sum(-1, keepdim=True)) + top  # 64 bits: x - top is
    # a beam's best: the order of its scores is that of its logits, ties to the lowest token
    index = torch.arange(vocab, device="cuda")
    keys = torch.where(x > -INF, _order(x) * (1 << 20) + ((1 << 20) - 1 - index), -1 << 60)
    best = keys.topk(min(width, vocab), dim=-1).values
    token = torch.where(best > -1 << 60, ((1 << 20) - 1) - (best & ((1 << 20) - 1)), 0)
    score = s["scores"].double()[:, None] + (x.gather(1, token).double() - lse)
    if s["done"] is not None:
        one = s["done"][:, None] & (torch.arange(token.shape[1], device="cuda") == 0)
        token = torch.where(one, s["pad_id"], token)
        score = torch.where(s["done"][:, None],
                            torch.where(one, s["scores"].double()[:, None], -INF), score)
        best = torch.where(one, 0, best)
    alive = (best > -1 << 60) & (s["scores"][:, None] > -INF)
    score = torch.where(alive, score, -INF).view(-1, beams * token.shape[1])
    at = score.sort(dim=-1, descending=True, stable=True)
    pick, score = at.indices[:, :width], at.values[:, :width]
    parent = (torch.arange(pick.shape[0], device="cuda")[:, None] * beams
              + pick // token.shape[1])
    token = token.view(pick.shape[0], -1).gather(1, pick)
    none = score == -INF
    out = [torch.where(none, -1, parent).to(torch.int32), torch.where(none, -1, token),
           score.float()]
    return [torch.nn.functional.pad(t, (0, width - t.shape[1]), value=v)
            for t, v in zip(out, (-1, -1, -INF))]


def _listings(table, listed, blocks):
    """How often each page is listed where `listed`."""
    page = torch.where(listed & (table >= 0), table.long(), blocks)
    return torch.zeros(blocks + 1, dtype=torch.int64, device="cuda").scatter_add_(
        0, page.flatten(), torch.ones_like(page).flatten())[:blocks]


def _compress(flags, size, descending=False):
    """The indices where `flags`, in order, then -1; and their number."""
    where = torch.arange(flags.numel(), device="cuda")
    rank = torch.cumsum(flags.long(), 0)
    count = rank[-1:]
    rank = count - rank if descending else rank - 1
    out = torch.full((size + 1,), -1, dtype=torch.int64, device="cuda")
    out.scatter_(0, torch.where(flags & (rank < size), rank, size), torch.where(flags, where, -1))
    return out[:size], count


def _move(caches, pairs):
    pairs = pairs[pairs[:, 1] >= 0].long()
    caches[:, :, pairs[:, 1]] = caches[:, :, pairs[:, 0]]


def _plain_fork(s):
    bs, blocks, table = s["bs"], s["blocks"], s["table"]
    rows, width = table.shape
    par = s["parents"].long()
    ok = (par >= 0) & (par < rows)
    par = par.clamp(0, rows - 1)
    pages = s["num_pages"].long().clamp(0, width)
    lens = torch.minimum(s["lens"].long().clamp(min=0), pages * bs)
    kept = (lens + bs - 1) // bs
    children = torch.zeros(rows, dtype=torch.int64, device="cuda").scatter_add_(0, par, ok.long())
    col = torch.arange(width, device="cuda")[None]
    live = _listings(table, (col < kept[:, None]) & (children > 0)[:, None], blocks)
    # a partial last page stays with its row's first child if no other row lists it
    order = torch.arange(rows, device="cuda")
    first = torch.full((rows,), rows, dtype=torch.int64, device="cuda").scatter_reduce_(
        0, par, torch.where(ok, order, rows), "amin")
    new_kept = torch.where(ok, kept[par], 0)
    new_lens = torch.where(ok, lens[par], 0)
    tail = (new_kept - 1).clamp(min=0)
    page = table[par, tail].long()
    copy = ((new_lens % bs != 0) & (page >= 0)
            & ((first[par] != order) | (live[page.clamp(min=0)] > 1)))
    taken = torch.cumsum(copy.long(), 0)
    count = s["free_count"].long()
    at = count - taken
    got = copy & (at >= 0)
    dst = torch.where(got, s["free_pages"][at.clamp(min=0)].long(), -1)
    new_pages = torch.where(copy & ~got, tail, new_kept)
    new_lens = torch.where(copy & ~got, tail * bs, new_lens)
    new = torch.where(col < new_kept[:, None], table[par], -1)
    new = torch.where(copy[:, None] & (col == tail[:, None]), dst.to(torch.int32)[:, None], new)
    copies = torch.stack((torch.where(got, page, -1), dst), 1)
    left = count - torch.minimum(taken[-1:], count)
    listed = _listings(table, col < pages[:, None], blocks) > 0
    freed = listed & (_listings(new, col < new_pages[:, None], blocks) == 0)
    free, more = _compress(freed, blocks)
    i = torch.arange(blocks, device="cuda")
    free = torch.where(i < left, s["free_pages"].long(),
                       torch.where(i < left + more, free[(i - left).clamp(min=0)], -1))
    _move(s["caches"], copies)
    return [new.to(torch.int32), new_pages.to(torch.int32), new_lens.to(torch.int32),
            free.to(torch.int32), (left + more).to(torch.int32), copies.to(torch.int32),
            s["caches"]]


def _plain_compact(s):
    blocks, table = s["blocks"], s["table"]
    col = torch.arange(table.shape[1], device="cuda")[None]
    held = col < s["num_pages"][:, None]
    used = _listings(table, held, blocks) > 0
    total = used.sum()
    page = torch.arange(blocks, device="cuda")
    src, _ = _compress(used & (page >= total), blocks // 2)
    dst, _ = _compress(~used & (page < total), blocks // 2)
    dst = torch.where(src >= 0, dst, -1)
    to = torch.cat((page, page[:1] - 1)).scatter_(0, torch.where(src >= 0, src, blocks), dst)
    new = torch.where(held & (table >= 0), to[table.clamp(min=0).long()], -1).to(torch.int32)
    free = torch.where(page < blocks - total, blocks - 1 - page, -1).to(torch.int32)
    moves = torch.stack((src, dst), 1).to(torch.int32)
    _move(s["caches"], moves)
    return [new, free, (blocks - total).view(1).to(torch.int32), moves, s["caches"]]


_PLAIN = {"attend": _plain_attend, "write": _plain_write, "beams": _plain_beams,
          "fork": _plain_fork, "compact": _plain_compact}
_OWN = {"attend": _own_attend, "write": _own_write, "beams": _own_beams, "fork": _own_fork,
        "compact": _own_compact}


# --------------------------------------------------------------------- work
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "attend":
        n = _spread(case["seqs"], case["lo"], case["hi"], 1)
        ctx = _spread(case["seqs"], case["ctx_lo"], case["ctx_hi"], 2)
        hd, n_q = case["hd"], case["n_q"]
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, ctx))
        tokens = sum(n) + sum(ctx)
        return dict(bytes=4 * sum(n) * n_q * hd + 2 * tokens * case["n_kv"] * (hd // 2 + hd // 16),
                    flops=4 * pairs * n_q * hd)
    if kind == "write":
        per = case["n_kv"] * case["hd"]  # a token's values, of K and of V
        t = case["tokens"]
        # 16 bits in, 4.5 out; the values in 32 bits (4.5 in, as they were just written)
        return dict(bytes=2 * t * per * (2 + 0.5625) + 2 * t * per * 0.5625
                    + 2 * (t + case["pad"]) * per * 4 + 8 * (t + case["pad"]),
                    flops=2 * t * per * 5)
    if kind == "beams":
        rows = case["seqs"] * case["beams"]
        values = rows * case["vocab"] * (1 - case["done"])
        return dict(bytes=values * (4 if case["wide"] else 2) + 5 * rows
                    + 16 * case["seqs"] * case["width"], flops=4 * values)
    page = 4 * case["layers"] * case["bs"] * case["n_kv"] * case["hd"]  # K and V, all layers
    if kind == "fork":
        lens, bs = _fork_lens(case), case["bs"]
        entries = sum(-(-x // bs) for x in lens)
        # of b draws of a parent (the lower of two uniform ones) some repeat
        b = case["beams"]
        repeats = b - sum(1 - (1 - (2 * (b - i) - 1) / b ** 2) ** b for i in range(b))
        copies = repeats * sum(1 for x in lens[::b] if x % bs)
        return dict(bytes=8 * entries + 32 * len(lens) + 2 * copies * page, flops=entries)
    held = [-(-x // case["bs"]) for x in _spread(case["seqs"], case["lo"], case["hi"], 1)]
    used = sum(held)
    blocks = used + case["spare"]
    moves = used * case["spare"] / blocks  # of a pool in random order
    return dict(bytes=8 * used + 4 * blocks + 8 * moves + 2 * moves * page, flops=used)


# -------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    """From the definitions: one sequence and head, row or page at a time."""
    s = _PREPARE[case["kind"]](case, seed)
    return _EXACT[case["kind"]](case, s)


def _half_bytes(p):
    return torch.stack((p.bitwise_and(15), p.bitwise_right_shift(4)), -1).reshape(*p.shape[:-1], -1)


def _decode(codes, scales, i, hd):
    """Channel by channel, in 64 bits: [..., hd / 2] bytes and their scales."""
    c = _half_bytes(codes).double() - 8
    where = []
    for ch in range(hd):
        b, r = divmod(ch, 32)
        dword = (r // 8) * (hd // 32) + b
        where.append(8 * dword + (r % 8) // 2 + 4 * (r % 2) if i == 0 else ch)
    return c[..., where] * scales.double().repeat_interleave(32, -1)


def _exact_attend(case, s):
    n = _spread(case["seqs"], case["lo"], case["hi"], 1)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    hd, bs, group = case["hd"], case["bs"], case["n_q"] // case["n_kv"]
    row = 0
    for r, a in enumerate(n):
        length = int(s["lens"][r])
        pages = s["table"][r, :-(-length // bs)].long()
        k, v = (_decode(s["codes"][i][pages], s["scales"][i][pages], i, hd).transpose(0, 1)
                .reshape(case["n_kv"], -1, hd)[:, :length] for i in range(2))
        last = torch.arange(length - a, length, device="cuda")
        for h in range(case["n_q"]):
            w = (s["q"][row:row + a, h].double() @ k[h // group].transpose(0, 1)) * s["scale"]
            w[torch.arange(length, device="cuda")[None] > last[:, None]] = -INF
            out[row:row + a, h] = torch.softmax(w, dim=1) @ v[h // group]
        row += a
    return out


def _exact_write(case, s):
    out = []
    for x in (s["key"], s["value"]):
        b = x.double().reshape(-1, 32)
        m = b[torch.arange(b.shape[0], device="cuda"), b.abs().argmax(1)]
        d = (m / -8).to(torch.float16).double()[:, None]
        q = torch.floor((b + 8.5 * d) / d).clamp(0, 15)
        v = torch.where(d == 0, 0.0, d * (q - 8)).reshape(x.shape)
        v[s["slots"] < 0] = 0
        out.append(v)
    return out


def _exact_beams(case, s):
    beams, width = case["beams"], case["width"]
    vocab = case["vocab"]
    parents, tokens, scores = [], [], []
    for i in range(case["seqs"]):
        rows = slice(i * beams, (i + 1) * beams)
        lp = torch.log_softmax(s["logits"][rows].double(), -1)
        total = s["scores"][rows].double()[:, None] + lp
        total[lp.isnan()] = -INF
        if s["done"] is not None:
            d = s["done"][rows]
            total[d] = -INF
            total[d, s["pad_id"]] = s["scores"][rows][d].double()
        flat = total.flatten()
        least = flat.topk(min(width, flat.numel())).values[-1]
        at = torch.nonzero((flat >= least) & (flat > -INF)).flatten()
        at = at[flat[at].sort(descending=True, stable=True).indices][:width]
        none = [-1] * (width - at.numel())
        parents.append((i * beams + at // vocab).tolist() + none)
        tokens.append((at % vocab).tolist() + none)
        scores.append(flat[at].tolist() + [-INF] * len(none))
    return [torch.tensor(parents, dtype=torch.int32), torch.tensor(tokens),
            torch.tensor(scores, dtype=torch.float64)]


def _exact_fork(case, s):
    bs = case["bs"]
    table, par = s["table"].tolist(), s["parents"].tolist()
    pages, lens = s["num_pages"].tolist(), s["lens"].tolist()
    free = s["free_pages"].tolist()[:int(s["free_count"])]
    before = {p for r, n in zip(table, pages) for p in r[:n]}
    live = {}
    for r in sorted(set(par)):
        for p in table[r][:-(-lens[r] // bs)]:
            live[p] = live.get(p, 0) + 1
    new, new_pages, new_lens, copies, had = [], [], [], [], set()
    for r in par:
        row = table[r][:-(-lens[r] // bs)]
        length, pair = lens[r], [-1, -1]
        if length % bs and (r in had or live[row[-1]] > 1):
            if free:
                pair = [row[-1], free.pop()]
                row[-1] = pair[1]
            else:
                row.pop()
                length = len(row) * bs
        had.add(r)
        copies.append(pair)
        new.append(row + [-1] * (len(table[0]) - len(row)))
        new_pages.append(len(row))
        new_lens.append(length)
    free += sorted(before - {p for r in new for p in r})
    for src, dst in copies:
        if dst >= 0:
            s["caches"][:, :, dst] = s["caches"][:, :, src]
    out = [new, new_pages, new_lens, free + [-1] * (s["blocks"] - len(free)), [len(free)], copies]
    return [torch.tensor(x, dtype=torch.int32) for x in out] + [s["caches"]]


def _exact_compact(case, s):
    blocks = s["blocks"]
    table, pages = s["table"].tolist(), s["num_pages"].tolist()
    used = sorted({p for r, n in zip(table, pages) for p in r[:n]})
    holes = sorted(set(range(len(used))) - set(used))
    moves = [[p, holes[i]] for i, p in enumerate(p for p in used if p >= len(used))]
    to = {p: p for p in used} | {a: b for a, b in moves}
    new = [[to[p] for p in r[:n]] + [-1] * (len(r) - n) for r, n in zip(table, pages)]
    for a, b in moves:
        s["caches"][:, :, b] = s["caches"][:, :, a]
    free = list(range(blocks - 1, len(used) - 1, -1))
    out = [new, free + [-1] * len(used), [len(free)],
           moves + [[-1, -1]] * (blocks // 2 - len(moves))]
    return [torch.tensor(x, dtype=torch.int32) for x in out] + [s["caches"]]


_EXACT = {"attend": _exact_attend, "write": _exact_write, "beams": _exact_beams,
          "fork": _exact_fork, "compact": _exact_compact}
