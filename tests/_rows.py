"""Float64 references of the row attentions and of the request tables, and
tolerances derived from the roundings that the kernels document."""
from __future__ import annotations

import numpy as np
import torch

# Half a step of bf16 relative to the value.  A row's output is rounded once
# (U |out|), and each probability once before it multiplies V (at most U sum p |v|).
U = 2.0 ** -8
# What fp32 adds, relative to sum p |v|: a score is a sum of up to 128 exact
# products in fp32 (off by at most 128 * 2^-24 * sum |q k|; sum |q k| * scale is
# below 2^5 for the inputs here, N(0, 1) of up to 128 dims, in 2^-24 * 2^12 =
# 2^-12 of p), the exponent's argument and exp2 a few 2^-24 of magnitudes below
# 2^7, the sums over at most 2^14 tokens are of blocks of 64 and below that.
FP32 = 2.0 ** -11


def attend64(q, k, v, scale, seen):
    """q [rows, n_q, hd], k / v [tokens, n_kv, hd] float64, seen [rows, tokens]
    -> (out, sum p |v|) [rows, n_q, hd]; a row that sees nothing is 0."""
    n_q, n_kv = q.shape[1], k.shape[1]
    kk = k.repeat_interleave(n_q // n_kv, 1)
    vv = v.repeat_interleave(n_q // n_kv, 1)
    s = torch.einsum("rhd,thd->hrt", q, kk) * scale
    s = torch.where(seen[None], s, -torch.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e300)
    p = torch.exp(s - top)
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot > 0, tot, 1.0)
    return torch.einsum("hrt,thd->rhd", p, vv), torch.einsum("hrt,thd->rhd", p, vv.abs())


def gather(cache, table, n):
    """The first n tokens of a sequence: cache [blocks, bs, n_kv, hd]."""
    bs = cache.shape[1]
    pages = table[: -(-n // bs)].long()
    return cache[pages].reshape(-1, *cache.shape[2:])[:n].double()


def prompt64(q, k, v, table, start, lens, scale):
    """(out, sum p |v|, row is of a sequence), everything on the CPU."""
    cap = table.shape[1] * k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    mine = torch.zeros(q.shape[0], dtype=torch.bool)
    for r in range(len(lens)):
        a, b = min(int(start[r]), q.shape[0]), min(int(start[r + 1]), q.shape[0])
        if b <= a:
            continue
        mine[a:b] = True
        L = min(max(int(lens[r]), 0), cap)
        if L == 0:
            continue
        pos = torch.arange(L - (b - a), L)
        seen = torch.arange(L)[None] <= pos[:, None]
        out[a:b], mag[a:b] = attend64(q[a:b].double(), gather(k, table[r], L),
                                      gather(v, table[r], L), scale, seen)
    return out, mag, mine


def prefix64(q, k, v, ptable, prefix, table, lens, scale):
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    bs = k.shape[1]
    prefix = min(max(prefix, 0), ptable.numel() * bs)
    for r in range(q.shape[0]):
        L = min(max(int(lens[r]), 0), table.shape[1] * bs) if int(lens[r]) > prefix else max(
            int(lens[r]), 0)
        t = torch.arange(L)
        page = torch.where(t < prefix, ptable[(t // bs).clamp(max=ptable.numel() - 1)],
                           table[r][(t // bs).clamp(max=table.shape[1] - 1)]).long()
        if L == 0:
            continue
        kk, vv = k[page, t % bs].double(), v[page, t % bs].double()
        out[r:r + 1], mag[r:r + 1] = attend64(q[r:r + 1].double(), kk, vv, scale,
                                              torch.ones((1, L), dtype=torch.bool))
    return out, mag


def assert_rows(got, ref, mag, what=""):
    """|got - ref| <= U |ref| + (U + FP32) sum p |v|, element-wise (see above)."""
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bound = U * ref.abs() + (U + FP32) * mag + 1e-30
    over = ((got - ref).abs() / bound).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.3g} of the bound"


def tables64(query, context, held, free, count, table, bs, max_tokens):
    """request_tables token by token (lists and numpy on the host)."""
    table, held = np.array(table), list(held)
    width = table.shape[1]
    left = list(free[:count])
    pos, slot, start, lens = [], [], [0], []
    for r, (n, c) in enumerate(zip(query, context)):
        n = max(n, 0)
        want = min(-(-(n + c) // bs), width)
        b = held[r]
        while b < want:
            if left:
                table[r, b] = left.pop()
                held[r] += 1
            else:
                table[r, b] = -1
            b += 1
        for t in range(c, c + n):
            pos.append(t)
            pg = table[r, t // bs] if t // bs < width else -1
            slot.append(int(pg) * bs + t % bs if pg >= 0 else -1)
        start.append(start[-1] + n)
        lens.append(c + n)
    pad = max_tokens - len(pos)
    return (table, held, len(left), start, lens, (pos + [0] * pad)[:max_tokens],
            (slot + [-1] * pad)[:max_tokens])
