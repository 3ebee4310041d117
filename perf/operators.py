"""What a serving step does with prompts, shared prefixes and the paged cache's
tables, as cases that can be timed and checked:

  prompt   causal attention of packed query rows over the paged cache: whole
           prompts, chunks behind a context, a few drafted tokens a sequence
  prefix   decode attention of a batch whose sequences share a prefix
  tables   block tables, slots, positions and offsets from request lengths

  listed()             the cases, dicts of plain values
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  inputs on the GPU, from the seed
  run(state)           one pass: the plain form, or with `own` the framework's call
  work(case)           bytes and flops that the pass cannot do without
  exact(case, seed)    the outputs in 64 bits, written apart from the plain form

Shapes are the 4B decoder's (32 q / 8 kv heads of 128, pages of 128 tokens,
contexts to 32768) and generic ones: heads of 64, other groups, odd lengths,
pages of 32 and 64.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16


# --------------------------------------------------------------------- cases
def _prompt(name, seqs, lo, hi, ctx_lo, ctx_hi, n_q=32, n_kv=8, hd=128, bs=128, pad=0):
    return dict(name=name, kind="prompt", seqs=seqs, lo=lo, hi=hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
                n_q=n_q, n_kv=n_kv, hd=hd, bs=bs, pad=pad)


def _prefix(name, seqs, prefix, lo, hi, n_q=32, n_kv=8, hd=128, bs=128):
    return dict(name=name, kind="prefix", seqs=seqs, prefix=prefix, lo=lo, hi=hi, n_q=n_q,
                n_kv=n_kv, hd=hd, bs=bs)


def _tables(name, seqs, lo, hi, ctx_lo, ctx_hi, bs=128, pad=0):
    return dict(name=name, kind="tables", seqs=seqs, lo=lo, hi=hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
                bs=bs, pad=pad)


def listed() -> list[dict]:
    return [
        # a short question to a fresh session: the smallest prompt, latency
        _prompt("prompt_17", 1, 17, 17, 0, 0),
        # one prompt of ordinary length
        _prompt("prompt_2048", 1, 2048, 2048, 0, 0),
        # ragged prompts packed into one pass whose buffers are padded
        _prompt("prompt_packed", 12, 1, 1500, 0, 0, pad=37),
        # the longest prompt in one pass
        _prompt("prompt_8192", 1, 8192, 8192, 0, 0),
        # one chunk of a long prompt, behind what earlier chunks left in the cache
        _prompt("chunk_behind_16k", 1, 509, 509, 16000, 16000),
        # drafted tokens of eight sequences, verified in one pass
        _prompt("drafts_8seq", 8, 5, 5, 300, 8000),
        # another layout: heads of 64, seven q heads a kv head, pages of 32
        _prompt("prompt_hd64", 5, 3, 1111, 0, 700, n_q=14, n_kv=2, hd=64, bs=32, pad=5),
        # a chat batch under one system prompt
        _prefix("prefix_8seq", 8, 4096, 1, 512),
        # a large batch under a long document, whose end is inside a page
        _prefix("prefix_64seq", 64, 32700, 100, 2048),
        # another layout, a short prefix
        _prefix("prefix_hd64", 3, 300, 1, 90, n_q=16, n_kv=4, hd=64, bs=64),
        # one decode step of a batch: a new page now and then
        _tables("tables_decode", 16, 1, 1, 1, 6000),
        # a prefill step of many requests
        _tables("tables_prompts", 256, 1, 512, 0, 2000, pad=100),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8, 128), (32, 8, 128), (32, 8, 128), (16, 16, 128), (14, 2, 64), (24, 8, 64),
          (40, 8, 128), (8, 1, 128), (16, 4, 64)]


def draw(rng) -> dict:
    kind = rng.choice(["prompt", "prompt", "prompt", "prefix", "prefix", "tables"])
    n_q, n_kv, hd = rng.choice(_HEADS)
    bs = rng.choice([32, 64, 128, 128, 256])
    if kind == "prompt":
        seqs = _log_int(rng, 1, 32)
        most = 8192 * 8192 * 32 // max(n_q, 32)  # scores a head: no more than the longest prompt
        hi = _log_int(rng, 1, math.isqrt(most) // seqs)
        lo = rng.choice([1, hi, max(1, hi // 8)])
        ctx = rng.choice([0, 0, _log_int(rng, 1, 16384)])
        ctx = min(ctx, most // (seqs * seqs * hi) - hi)
        c = _prompt("", seqs, lo, hi, ctx // rng.choice([1, 3]), ctx, n_q, n_kv, hd, bs,
                    rng.choice([0, 0, 3, 64]))
    elif kind == "prefix":
        seqs = _log_int(rng, 2, 64)
        prefix = _log_int(rng, 32, 32768)
        hi = _log_int(rng, 1, 2048)
        c = _prefix("", seqs, prefix, rng.choice([1, hi]), hi, n_q, n_kv, hd, bs)
    else:
        seqs = _log_int(rng, 1, 512)
        hi = _log_int(rng, 1, max(1, 131072 // seqs))
        ctx = _log_int(rng, 1, 4096)
        c = _tables("", seqs, 1, hi, 0, ctx, bs, rng.choice([0, 17, 500]))
    del c["name"]
    return c


# -------------------------------------------------------------------- inputs
def _gen(seed: int, salt: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) & 0x7FFFFFFF) * 1000003 + salt)
    return g


def _spread(n: int, lo: int, hi: int, salt: int) -> list[int]:
    """n lengths from lo to hi, both among them where n allows, spread over
    their logarithm; the same for every seed, so that a case is one amount of
    work."""
    r = random.Random(1000003 * n + 8191 * lo + 31 * hi + salt)
    out = [hi] + [min(hi, max(lo, _log_int(r, max(lo, 1), max(hi, 1)))) for _ in range(n - 2)]
    out += [lo] if n > 1 else []
    r.shuffle(out)
    return out


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(query lengths, lengths in the cache before them)"""
    return (_spread(case["seqs"], case["lo"], case["hi"], 1),
            _spread(case["seqs"], case["ctx_lo"], case["ctx_hi"], 2))


def _i32(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(case, seed, blocks):
    g = _gen(seed, 1)
    shape = (blocks, case["bs"], case["n_kv"], case["hd"])
    return [torch.empty(shape, dtype=BF16, device="cuda").normal_(0.0, 1.0, generator=g)
            for _ in range(2)]


def prepare(case: dict, seed: int) -> dict:
    s = _PREPARE[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    if own:
        s["ops"] = ops = _ops()
        if case["kind"] == "prompt":
            s["workspace"] = ops.prompt_attention_workspace(s["q"], s["k"], s["table"])
        elif case["kind"] == "prefix":
            s["workspace"] = ops.shared_prefix_attention_workspace(s["q"], s["k"],
                                                                   s["prefix_table"], s["table"])
        else:
            s["out"] = ops.request_tables_out(s["num_pages"], s["max_tokens"])
    return s


def _ops():
    import importlib
    import os

    os.environ.setdefault("SMX_ALLOW_UNVALIDATED", "1")  # the library as built is what is measured
    import __graft_entry__

    return importlib.import_module(__graft_entry__.load_package().__name__ + ".native.torch_ops")


def _prep_prompt(case, seed):
    n, ctx = _lengths(case)
    lens = [a + b for a, b in zip(n, ctx)]
    per_seq = -(-max(lens) // case["bs"]) + 1
    blocks = case["seqs"] * per_seq
    k, v = _cache(case, seed, blocks)
    table = torch.randperm(blocks, generator=_gen(seed, 2), device="cuda").to(torch.int32)
    rows = sum(n) + case["pad"]
    q = torch.randn((rows, case["n_q"], case["hd"]), generator=_gen(seed, 3), device="cuda")
    start = [0]
    for x in n:
        start.append(start[-1] + x)
    return dict(q=q.to(BF16), k=k, v=v, table=table.view(case["seqs"], per_seq),
                start=_i32(start), lens=_i32(lens), scale=1.0 / math.sqrt(case["hd"]),
                total=sum(n), live=sum(lens),
                out=torch.zeros((rows, case["n_q"], case["hd"]), dtype=BF16, device="cuda"))


def _prep_prefix(case, seed):
    suffix = _spread(case["seqs"], case["lo"], case["hi"], 3)
    bs, prefix = case["bs"], case["prefix"]
    lens = [prefix + x for x in suffix]
    shared = prefix // bs  # whole pages of the prefix; its tail is in every sequence's own page
    per_seq = -(-max(lens) // bs)
    blocks = shared + 1 + case["seqs"] * (per_seq - shared)
    k, v = _cache(case, seed, blocks)
    perm = torch.randperm(blocks, generator=_gen(seed, 2), device="cuda").to(torch.int32)
    prefix_table = perm[:shared + 1].contiguous()
    own_pages = perm[shared + 1:].view(case["seqs"], per_seq - shared)
    table = torch.cat((prefix_table[:shared].expand(case["seqs"], shared), own_pages), 1)
    q = torch.randn((case["seqs"], case["n_q"], case["hd"]), generator=_gen(seed, 3),
                    device="cuda")
    return dict(q=q.to(BF16), k=k, v=v, prefix_table=prefix_table, prefix_len=_i32([prefix]),
                prefix=prefix, table=table.contiguous(), lens=_i32(lens), suffix=_i32(suffix),
                live=sum(suffix), scale=1.0 / math.sqrt(case["hd"]))


def _prep_tables(case, seed):
    n, ctx = _lengths(case)
    bs = case["bs"]
    held = [-(-c // bs) for c in ctx]
    per_seq = -(-max(a + b for a, b in zip(n, ctx)) // bs) + 1
    need = sum(max(0, -(-(a + b) // bs) - h) for a, b, h in zip(n, ctx, held))
    blocks = sum(held) + need + 9
    perm = torch.randperm(blocks, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    col = torch.arange(per_seq, device="cuda")[None]
    h = _i32(held)[:, None]
    first = torch.cumsum(h, 0) - h
    table = torch.where(col < h, perm[(first + col).clamp(max=blocks - 1)], -1).to(torch.int32)
    return dict(query_lens=_i32(n), context_lens=_i32(ctx), num_pages=_i32(held),
                free_pages=perm[sum(held):].contiguous(), free_count=_i32([blocks - sum(held)]),
                table=table.contiguous(), bs=bs, max_tokens=sum(n) + case["pad"])


_PREPARE = {"prompt": _prep_prompt, "prefix": _prep_prefix, "tables": _prep_tables}


# ---------------------------------------------------------------------- run
def run(state: dict):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_prompt(s):
    return s["ops"].prompt_attention(s["q"], s["k"], s["v"], s["table"], s["start"], s["lens"],
                                     s["scale"], workspace=s["workspace"], out=s["out"])


def _own_prefix(s):
    return s["ops"].shared_prefix_attention(s["q"], s["k"], s["v"], s["prefix_table"],
                                            s["prefix_len"], s["table"], s["lens"], s["scale"],
                                            workspace=s["workspace"])


def _own_tables(s):
    r = s["ops"].request_tables(s["query_lens"], s["context_lens"], s["num_pages"],
                                s["free_pages"], s["free_count"], s["table"], s["bs"],
                                out=s["out"])
    return [s["table"], r.num_pages, r.free_count, r.query_start_loc, r.seq_lens, r.positions,
            r.slot_mapping]


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the tokens that a row sees: q [rows, n_q, hd],
    k and v [tokens, n_kv, hd], seen [rows, tokens]; a row that sees none is 0."""
    rows, n_q, hd = q.shape
    n_kv = k.shape[1]
    qf = q.float().view(rows, n_kv, n_q // n_kv, hd).permute(1, 2, 0, 3).reshape(n_kv, -1, hd)
    s = torch.matmul(qf, k.float().permute(1, 2, 0).contiguous()).mul_(scale)
    s = s.view(n_kv, n_q // n_kv, rows, -1).masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_kv, -1, k.shape[0]), v.float().permute(1, 0, 2).contiguous())
    o = o.view(n_kv, n_q // n_kv, rows, hd) / torch.where(total > 0, total, 1.0)
    return o.permute(2, 0, 1, 3).reshape(rows, n_q, hd).to(BF16)


def _tokens(cache, table, seq, pos):
    """The cache's rows of the tokens at positions `pos` of sequences `seq`."""
    bs = cache.shape[1]
    slot = table[seq, pos // bs].long() * bs + pos % bs
    return cache.view(-1, *cache.shape[2:])[slot]


def _ragged(lens, total):
    """(sequence, index within it) of `total` items of sequences of these lengths."""
    seq = torch.repeat_interleave(lens.long(), output_size=total)
    first = torch.cumsum(lens, 0) - lens
    return seq, torch.arange(total, device=lens.device) - first[seq]


def _plain_prompt(s):
    n = s["start"][1:] - s["start"][:-1]
    q_seq, q_at = _ragged(n, s["total"])
    q_pos = q_at + (s["lens"] - n)[q_seq]
    k_seq, k_pos = _ragged(s["lens"], s["live"])
    seen = (q_seq[:, None] == k_seq[None]) & (k_pos[None] <= q_pos[:, None])
    o = _attend(s["q"][:s["total"]], _tokens(s["k"], s["table"], k_seq, k_pos),
                _tokens(s["v"], s["table"], k_seq, k_pos), seen, s["scale"])
    out = torch.zeros_like(s["q"])
    out[:s["total"]] = o
    return out


def _plain_prefix(s):
    seqs, prefix = s["q"].shape[0], s["prefix"]
    p_pos = torch.arange(prefix, device="cuda")
    k_seq, k_pos = _ragged(s["suffix"], s["live"])
    k_pos = k_pos + prefix
    pt, zero = s["prefix_table"][None], torch.zeros_like(p_pos)
    k, v = (torch.cat((_tokens(c, pt, zero, p_pos), _tokens(c, s["table"], k_seq, k_pos)))
            for c in (s["k"], s["v"]))
    row = torch.arange(seqs, device="cuda")
    seen = torch.cat((torch.ones((seqs, prefix), dtype=torch.bool, device="cuda"),
                      row[:, None] == k_seq[None]), 1)
    return _attend(s["q"], k, v, seen, s["scale"])


def _plain_tables(s):
    bs, table, pages = s["bs"], s["table"], s["num_pages"].long()
    width = table.shape[1]
    n = s["query_lens"].long()
    lens = s["context_lens"].long() + n
    want = torch.clamp((lens + bs - 1) // bs, max=width)
    need = torch.clamp(want - pages, min=0)
    first = torch.cumsum(need, 0) - need
    count = s["free_count"].long()
    col = torch.arange(width, device="cuda")[None]
    fresh = (col >= pages[:, None]) & (col < (pages + need)[:, None])
    at = count - 1 - (first[:, None] + col - pages[:, None])
    page = torch.where(at >= 0, s["free_pages"][at.clamp(0, s["free_pages"].numel() - 1)], -1)
    table = torch.where(fresh, page, table).to(torch.int32)
    got = torch.minimum(need, torch.clamp(count - first, min=0))
    start = torch.cat((torch.zeros_like(count), torch.cumsum(n, 0)))
    tok = torch.arange(s["max_tokens"], device="cuda")
    seq = torch.searchsorted(start[1:], tok, right=True)
    real = seq < n.numel()
    seq = seq.clamp(max=n.numel() - 1)
    pos = torch.where(real, s["context_lens"][seq] + tok - start[seq], 0)
    block = pos // bs
    page = table[seq, block.clamp(max=width - 1)].long()
    slot = torch.where(real & (block < width) & (page >= 0), page * bs + pos % bs, -1)
    return [table, (pages + got).to(torch.int32),
            torch.clamp(count - need.sum(), min=0).to(torch.int32), start.to(torch.int32),
            lens.to(torch.int32), pos, slot]


_PLAIN = {"prompt": _plain_prompt, "prefix": _plain_prefix, "tables": _plain_tables}
_OWN = {"prompt": _own_prompt, "prefix": _own_prefix, "tables": _own_tables}


# --------------------------------------------------------------------- work
def work(case: dict) -> dict:
    if case["kind"] == "tables":
        n, ctx = _lengths(case)
        bs = case["bs"]
        fresh = sum(max(0, -(-(a + b) // bs) - -(-b // bs)) for a, b in zip(n, ctx))
        tokens = sum(n) + case["pad"]
        # three lengths in, pages taken, three numbers and two 8-byte rows out
        return dict(bytes=4 * (3 * len(n) + 2 * fresh + 3 * len(n) + 3) + 16 * tokens,
                    flops=tokens + 4 * len(n))
    n_q, n_kv, hd = case["n_q"], case["n_kv"], case["hd"]
    if case["kind"] == "prompt":
        n, ctx = _lengths(case)
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, ctx))
        rows, tokens = sum(n), sum(n) + sum(ctx)
    else:
        suffix = _spread(case["seqs"], case["lo"], case["hi"], 3)
        rows, tokens = case["seqs"], case["prefix"] + sum(suffix)
        pairs = rows * case["prefix"] + sum(suffix)
    return dict(bytes=2 * hd * (2 * rows * n_q + 2 * tokens * n_kv), flops=4 * pairs * n_q * hd)


# -------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    """From the definition, in 64 bits: one sequence and one head at a time;
    the tables token by token on the host."""
    s = _PREPARE[case["kind"]](case, seed)
    return _EXACT[case["kind"]](case, s)


def _softmax_v(q, k, v, scale, last):
    """q [rows, hd] against k, v [tokens, hd]; row i sees the tokens 0..last[i]."""
    w = (q @ k.transpose(0, 1)) * scale
    beyond = torch.arange(k.shape[0], device=q.device).unsqueeze(0) > last.unsqueeze(1)
    w[beyond] = -math.inf
    return torch.softmax(w, dim=1) @ v


def _linear_cache(cache, pages, length):
    return cache[pages.long()].flatten(0, 1)[:length].double()


def _exact_prompt(case, s):
    n, ctx = _lengths(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["n_q"] // case["n_kv"]
    row = 0
    for r, (a, b) in enumerate(zip(n, ctx)):
        k = _linear_cache(s["k"], s["table"][r], a + b)
        v = _linear_cache(s["v"], s["table"][r], a + b)
        last = torch.arange(b, a + b, device="cuda")
        for h in range(case["n_q"]):
            out[row:row + a, h] = _softmax_v(s["q"][row:row + a, h].double(), k[:, h // group],
                                             v[:, h // group], s["scale"], last)
        row += a
    return out


def _exact_prefix(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["n_q"] // case["n_kv"]
    shared = case["prefix"]
    kp = _linear_cache(s["k"], s["prefix_table"], shared)
    vp = _linear_cache(s["v"], s["prefix_table"], shared)
    for r, x in enumerate(_spread(case["seqs"], case["lo"], case["hi"], 3)):
        k = torch.cat((kp, _linear_cache(s["k"], s["table"][r], shared + x)[shared:]))
        v = torch.cat((vp, _linear_cache(s["v"], s["table"][r], shared + x)[shared:]))
        last = torch.full((group,), shared + x - 1, device="cuda")
        for h in range(case["n_kv"]):
            rows = slice(h * group, (h + 1) * group)
            out[r, rows] = _softmax_v(s["q"][r, rows].double(), k[:, h], v[:, h], s["scale"],
                                      last)
    return out


def _exact_tables(case, s):
    n, ctx = _lengths(case)
    bs = case["bs"]
    table = s["table"].tolist()
    free = s["free_pages"].tolist()[:int(s["free_count"])]
    held = s["num_pages"].tolist()
    positions, slots, start, lens = [], [], [0], []
    for r in range(len(n)):
        while held[r] * bs < n[r] + ctx[r]:
            table[r][held[r]] = free.pop()
            held[r] += 1
        for t in range(ctx[r], ctx[r] + n[r]):
            positions.append(t)
            slots.append(table[r][t // bs] * bs + t % bs)
        start.append(len(positions))
        lens.append(ctx[r] + n[r])
    pad = s["max_tokens"] - len(positions)
    out = [table, held, [len(free)], start, lens, positions + [0] * pad, slots + [-1] * pad]
    kinds = [torch.int32] * 5 + [torch.int64] * 2
    return [torch.tensor(x, dtype=d) for x, d in zip(out, kinds)]


_EXACT = {"prompt": _exact_prompt, "prefix": _exact_prefix, "tables": _exact_tables}
