"""Attention over a KV cache held in 4 bits, token by token: V has one dim of a token that is
not 0, so that a row's output in a dim is the weights of a few tokens, each of which a
dropped, doubled or misplaced one would change by much more than the roundings do."""
import math

import pytest
import torch

from _rows import FP32, U, prompt64
from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16

CASES = [
    # n, ctx, n_q, n_kv, hd, bs, prompts
    ([1, 1, 1], [0, 700, 95], 32, 8, 128, 32, False),
    ([1, 1], [1000, 300], 14, 2, 64, 64, False),
    ([5, 1, 17], [640, 0, 90], 16, 4, 128, 128, False),
    ([64, 100, 3], [0, 333, 1900], 32, 8, 128, 32, True),
    ([450], [0], 32, 8, 128, 64, True),
    ([310, 77], [31, 500], 40, 8, 128, 128, True),
    ([200, 1, 450], [64, 2000, 0], 16, 4, 64, 32, True),
    ([500], [300], 28, 4, 64, 128, True),
    ([40, 40, 40, 40, 0, 1], [1200, 0, 50, 64, 0, 9], 64, 16, 64, 64, True),
    ([1, 600], [0, 40], 16, 1, 128, 256, True),
    ([1500], [0], 16, 4, 64, 64, True),
    ([300], [3000], 32, 8, 128, 64, True),
    ([2100], [0], 32, 8, 128, 32, True),
    ([2100], [0], 32, 8, 128, 128, True),
    ([2100], [0], 32, 8, 64, 32, True),
    ([300, 290, 310], [900, 0, 33], 32, 8, 64, 64, True),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_every_token_has_its_weight(case):
    """Against attention in 64 bits over the values that the kernels multiply: those of the
    cache, of prompts rounded to fp16.  So the outputs' rounding to bf16 and the weights' to
    fp16 (half a step is 2^-12) are left."""
    n, ctx, n_q, n_kv, hd, bs, prompts = case
    print(f"case {case}", flush=True)
    ops = pkg("native.torch_ops")
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = [a + b for a, b in zip(n, ctx)]
    per = -(-max(lens) // bs) + 1
    blocks = len(n) * per + 2
    cache = ops.q4_kv_cache(blocks, bs, n_kv, hd, "cuda")
    table = torch.randperm(blocks, generator=g, device="cuda")[:len(n) * per].to(
        torch.int32).view(len(n), per)
    for r, length in enumerate(lens):
        t = torch.arange(length, device="cuda")
        slots = table[r][t // bs].long() * bs + t % bs
        key = torch.randn((length, n_kv, hd), generator=g, device="cuda").to(BF16)
        value = torch.zeros((length, n_kv, hd), dtype=BF16, device="cuda")
        for h in range(n_kv):
            value[t, h, (5 * t + h) % hd] = 1 + 3 * torch.rand(
                length, generator=g, device="cuda").to(BF16)
        ops.reshape_and_cache_q4(key, value, cache, slots)
    q = torch.randn((sum(n), n_q, hd), generator=g, device="cuda").to(BF16)
    start = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32)
    lens = torch.tensor(lens, dtype=torch.int32)
    got = ops.q4_attention(q, cache, table, lens.cuda(), 1 / math.sqrt(hd),
                           query_start_loc=start.cuda())
    held = ops.q4_kv_read(cache, torch.arange(blocks * bs, device="cuda"))
    k, v = (x.view(blocks, bs, n_kv, hd) for x in held)
    if prompts:
        k, v = k.half(), v.half()
    ref, mag, mine = prompt64(q.cpu(), k.cpu(), v.cpu(), table.cpu(), start, lens,
                              1 / math.sqrt(hd))
    assert mine.all()
    over = (got.double().cpu() - ref).abs() / (U * ref.abs() + (2.0 ** -12 + FP32) * mag + 1e-30)
    assert over.max() <= 1.0, f"{case}: {over.max():.3g} of the bound"


def test_sequences_of_2_31_tokens():
    """Three of the longest tables, of one page again and again (K and V 0) but for a page at the
    front, in the middle or at the end, whose tokens have all the weight.  Parts of equal
    length would end past 2^31 tokens here."""
    ops = pkg("native.torch_ops")
    bs, hd, n_kv, width = 4096, 64, 4, 524286
    cache = ops.q4_kv_cache(2, bs, n_kv, hd, "cuda")
    ones = torch.ones((bs, n_kv, hd), dtype=BF16, device="cuda")
    ops.reshape_and_cache_q4(8 * ones, 3 * ones, cache, torch.arange(bs, 2 * bs, device="cuda"))
    table = torch.zeros((3, width), dtype=torch.int32, device="cuda")
    table[[0, 1, 2], [0, width // 2, width - 1]] = 1
    lens = torch.full((3,), width * bs, dtype=torch.int32, device="cuda")
    q = torch.ones((3, n_kv, hd), dtype=BF16, device="cuda")
    # scores 64 against 0: e^-64 2^31 / 4096 of the weight is elsewhere
    got = ops.q4_attention(q, cache, table, lens, hd ** -0.5)
    assert torch.equal(got, torch.full_like(got, 3.0))
