"""Few rows (decode steps, drafts) over a KV cache held in 4 bits: how exact they are, and values
of any size that the cache can hold."""
import math

import pytest
import torch

from _rows import FP32, U
from _util import pkg
from test_gpu_q4_prompt_range import F16, Rows

pytestmark = pytest.mark.gpu
CASES = [([1, 1, 1], [700, 95, 5000], 32, 8, 128, 32), ([1], [20000], 14, 2, 64, 64),
         ([5, 1, 17], [640, 20, 90], 16, 4, 128, 128), ([1] * 40, [37 * i for i in range(40)], 32, 8, 128, 64),
         ([1] * 20, [400 + 83 * i for i in range(20)], 16, 4, 64, 32), ([90], [0], 8, 2, 128, 32),
         ([1] * 3, [30, 300, 3000], 6, 6, 64, 4096)]


class Few(Rows):
    def grow(self):
        """V of a token 2^20 times that of one 2000 before: the limit of its scales rises."""
        for r, length in enumerate(self.lens):
            t = torch.arange(length, device="cuda")
            slots = self.table[r][t // self.bs].long() * self.bs + t % self.bs
            k, v = self.ops.q4_kv_read(self.cache, slots)
            v = v * 2.0 ** (t % 2000 / 100 - 12)[:, None, None]
            self.ops.reshape_and_cache_q4(k.bfloat16(), v.bfloat16(), self.cache, slots)

    def units(self):
        """sum p |d| of the rows, for every dim."""
        group = self.q.shape[1] // self.n_kv
        k = self.ops.q4_kv_read(self.cache, torch.arange(
            self.cache.num_blocks * self.bs, device="cuda"))[0].view(-1, self.bs, self.n_kv, self.hd)
        d = self.cache.scales[1].double().abs().repeat_interleave(32, -1).transpose(1, 2)
        outs = []
        for r, length in enumerate(self.lens):
            a, b = int(self.start[r]), int(self.start[r + 1])
            kk, dd = (x[self.table[r, :-(-length // self.bs)].long()].flatten(0, 1)[:length].double()
                      for x in (k, d))
            seen = torch.arange(length, device="cuda")[None] <= torch.arange(
                length - (b - a), length, device="cuda")[:, None]
            heads = []
            for h in range(self.q.shape[1]):
                s = torch.where(seen, self.q[a:b, h].double() @ kk[:, h // group].t() * self.hd ** -0.5,
                                -math.inf)
                heads.append(torch.softmax(s, -1) @ dd[:, h // group])
            outs.append(torch.stack(heads, 1))
        return torch.cat(outs)


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_the_outputs_rounding_is_what_counts(case):
    """N(0, 1): the weights' rounding to fp16, with V's scale, is an eighth of the outputs' own to
    bf16 and independent of it: together 1.01 times that alone, below 1.1."""
    c = Few(case, "plain")
    ref = c.reference()[0]
    own = (ref.bfloat16().double() - ref).norm()
    off = (c.run().double() - ref).norm()
    print(case, (off / ref.norm()).item(), (own / ref.norm()).item(), flush=True)
    assert off <= 1.1 * own


@pytest.mark.parametrize("kind", ["plain", "large", "small", "growing"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_values_of_any_size(case, kind):
    """Element by element: the outputs' rounding, the weights' and what fp32 adds (FP32), and to
    sums of weights times 16 + code (31 times V's scale, a thirty-first and more of |v| where a
    code is not 8): one for every 32 tokens of a wave and 8 to join.  A weight times its scale
    is held to 2^-36 of the largest weight times the largest scale, so to 2^-35 of it times |v|."""
    print(case, kind, flush=True)
    c = Few(case, "plain" if kind == "growing" else kind)
    if kind == "growing":
        c.grow()
    ref, mag, top = c.reference()
    assert top.max() < 40
    held = c.ops.q4_kv_read(c.cache, torch.arange(c.cache.num_blocks * c.bs, device="cuda"))
    most = held[1].abs().max().item()
    bound = U * ref.abs() + (F16 + FP32) * mag + max(c.lens) * 2.0 ** -35 * most + 1e-30
    if kind == "large":
        assert (c.cache.scales[0].float().abs() >= 2.0 ** 13).any()
        assert c.cache.scales[1].float().abs().max() == 65504 or max(c.lens) < 100
    # sums of weights times 31 scales, of which the codes' eights are taken off again
    chain = max(c.lens) / 32 + 8
    bound += 31 * 2.0 ** -23 * chain * c.units()
    got = c.run().double()
    assert torch.isfinite(got).all()
    over = ((got - ref).abs() / bound).max().item()
    assert over <= 1.0, f"{over:.3g} of the bound"


def test_decode_steps_of_many_heads_a_group():
    """Rows without offsets that go to the prompts' kernels, against the same with them."""
    c = Few(([1] * 40, [2500 + i for i in range(40)], 100, 1, 128, 64), "plain")
    lens = torch.tensor(c.lens, dtype=torch.int32).cuda()
    got = c.ops.q4_attention(c.q, c.cache, c.table, lens, c.hd ** -0.5)
    assert torch.equal(got, c.run())
    ref = c.reference()[0]
    assert (got.double() - ref).norm() <= 1.15 * (ref.bfloat16().double() - ref).norm()
