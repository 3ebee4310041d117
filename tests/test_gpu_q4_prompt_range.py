"""Prompts over a KV cache held in 4 bits: how exact they are, and values of any size that the
cache can hold, among them those that are too large for fp16, the kernels' type."""
import math

import pytest
import torch

from _rows import FP32, U
from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
F16 = 2.0 ** -12  # half a step of fp16, relative
CASES = [([450], [0], 32, 8, 128, 64), ([310, 77], [31, 500], 40, 8, 128, 128),
         ([300], [3000], 32, 8, 128, 32), ([2100], [0], 32, 8, 128, 128),
         ([1500], [0], 16, 4, 64, 64), ([2100], [0], 32, 8, 64, 32)]


class Rows:
    def __init__(self, case, kind, seed=4):
        n, ctx, n_q, n_kv, hd, self.bs = case
        self.ops, self.hd, self.n, self.n_kv = pkg("native.torch_ops"), hd, n, n_kv
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        some = lambda share, *s: torch.rand(s, generator=g, device="cuda") < share  # noqa: E731
        self.lens = [a + b for a, b in zip(n, ctx)]
        per = -(-max(self.lens) // self.bs) + 1
        blocks = len(n) * per + 2
        self.cache = self.ops.q4_kv_cache(blocks, self.bs, n_kv, hd, "cuda")
        self.table = torch.randperm(blocks, generator=g, device="cuda")[:len(n) * per].to(
            torch.int32).view(len(n), per)
        self.start = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32)
        q = rand(sum(n), n_q, hd)
        if kind == "large":
            q[..., :32] *= 2.0 ** -17
        elif kind == "small":
            q *= 2.0 ** 17
        self.q = q.to(BF16)
        for r, length in enumerate(self.lens):
            t = torch.arange(length, device="cuda")
            slots = self.table[r][t // self.bs].long() * self.bs + t % self.bs
            k, v = rand(length, n_kv, hd), rand(length, n_kv, hd)
            if kind == "large":
                # some tokens' K in its first 32 dims, V in any: up to the cache's largest and
                # beyond it
                k[..., :32] *= torch.where(some(0.05, length, n_kv, 1), 2.0 ** 16, 1.0)
                big = some(0.02, length, n_kv, hd // 32, 1).float().expand(-1, -1, -1, 32)
                v *= 1 + big.reshape(v.shape) * 2.0 ** torch.randint(
                    13, 22, v.shape, generator=g, device="cuda")
            elif kind == "small":
                k *= 2.0 ** -17
                v *= 2.0 ** -17
            self.ops.reshape_and_cache_q4(k.to(BF16), v.to(BF16), self.cache, slots)

    def run(self):
        return self.ops.q4_attention(
            self.q, self.cache, self.table, torch.tensor(self.lens, dtype=torch.int32).cuda(),
            self.hd ** -0.5, query_start_loc=self.start.cuda())

    def reference(self):
        """(out, sum p |v|, the largest scale sum |q k|) in 64 bits over the cache's values."""
        held = self.ops.q4_kv_read(self.cache, torch.arange(
            self.cache.num_blocks * self.bs, device="cuda"))
        k, v = (x.view(-1, self.bs, self.n_kv, self.hd).double() for x in held)
        group = self.q.shape[1] // self.n_kv
        outs = []
        for r, length in enumerate(self.lens):
            a, b = int(self.start[r]), int(self.start[r + 1])
            kk, vv = (x[self.table[r, :-(-length // self.bs)].long()].flatten(0, 1)[:length]
                      for x in (k, v))
            seen = torch.arange(length, device="cuda")[None] <= torch.arange(
                length - (b - a), length, device="cuda")[:, None]
            heads = []
            for h in range(self.q.shape[1]):
                x, y, z = self.q[a:b, h].double(), kk[:, h // group], vv[:, h // group]
                p = torch.softmax(torch.where(seen, x @ y.t() * self.hd ** -0.5, -math.inf), -1)
                top = torch.where(seen, x.abs() @ y.abs().t() * self.hd ** -0.5, 0.0).amax(-1)
                heads.append((p @ z, p @ z.abs(), top[:, None].expand(-1, self.hd)))
            outs.append([torch.stack(x, 1) for x in zip(*heads)])
        return [torch.cat(x) for x in zip(*outs)]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_the_outputs_rounding_is_what_counts(case):
    """N(0, 1): roundings to fp16, of K, V and the weights, are an eighth of the outputs' own to
    bf16 each, and independent of them: together 1.03 times those alone, below 1.15."""
    c = Rows(case, "plain")
    ref = c.reference()[0]
    own = (ref.to(BF16).double() - ref).norm()
    off = (c.run().double() - ref).norm()
    print(case, (off / ref.norm()).item(), (own / ref.norm()).item(), flush=True)
    assert off <= 1.15 * own


@pytest.mark.parametrize("kind", ["plain", "large", "small"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_values_of_any_size(case, kind):
    """Element by element: the outputs' rounding; the weights' and V's to fp16 and what fp32 adds
    (FP32); K's, which moves a score by F16 top at most, and a weight with the sum's change by
    expm1 of twice that.  Among 16 tokens with a value that is too large the others are
    held to 2^-20, and weights of a tile with such V to 2^-27 of the largest."""
    print(case, kind, flush=True)
    c = Rows(case, kind)
    ref, mag, top = c.reference()
    assert top.max() < 40
    bound = U * ref.abs() + (2 * F16 + FP32) * mag + torch.expm1(2 * F16 * top) * (mag + ref.abs())
    if kind == "large":
        scales = c.cache.scales.float()
        assert (scales[0].abs() >= 2.0 ** 13).any() and scales[1].abs().max() == 65504
        # (a K of 2^-20 off moves a score by 2^-20 scale sum |q|, below 2^-16 here)
        bound += torch.expm1(torch.tensor(2.0 ** -15).double()).item() * (mag + ref.abs())
        bound += 2.0 ** -20 + max(c.lens) * 2.0 ** -27 * 6
    got = c.run().double()
    assert torch.isfinite(got).all()
    over = ((got - ref).abs() / (bound + 1e-30)).max().item()  # (0 of 0 is within)
    assert over <= 1.0, f"{over:.3g} of the bound"


def test_rows_with_an_infinity_or_a_nan():
    """Of a query: its row is NaN, the others are what they are without."""
    c = Rows(CASES[1], "plain")
    clean = c.run()
    c.q[5, 3, 100] = math.inf
    c.q[200, 0, 1] = -math.inf
    c.q[350, 39, 127] = math.nan
    got = c.run()
    for row, head in ((5, 3), (200, 0), (350, 39)):
        assert got[row, head].isnan().all()
        got[row, head] = clean[row, head]
    assert torch.equal(got, clean)


def test_query_rows_of_any_size():
    """A row of queries times 2^100 or 2^-100 and scores that are the same: by its own power of
    two, taken back by the scale of another call."""
    c = Rows(CASES[0], "plain")
    want = c.run()
    lens = torch.tensor(c.lens, dtype=torch.int32).cuda()
    for power in (100, -100, 23, -37):
        got = c.ops.q4_attention((c.q.float() * 2.0 ** power).to(BF16), c.cache, c.table, lens,
                                 c.hd ** -0.5 * 2.0 ** -power, query_start_loc=c.start.cuda())
        assert torch.equal(got, want), power
