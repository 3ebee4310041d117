"""Beam search's selection where many logits are alike: the sums of exponentials are those of
64 bits, so that beams tie where they do by the definition and stand in its order where
their scores differ by less than fp32 can tell."""
import numpy as np
import pytest
import torch

from _util import pkg
from test_gpu_beam_select import check, reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
SHIFTS = [1.5, -3.25, 0.0, 12.0, 15.875, 17.0, 100.0, 0.0078125]


def _select(x, c, beams, width):
    return pkg("native.torch_ops").beam_select(x, c, beams, width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1000, 20011, 151936])
def test_unlike_constant_rows_tie(vocab, dtype):
    """A constant row's best is log(1 / vocab) whatever the constant: all beams tie."""
    print(vocab, dtype, flush=True)
    beams, width = len(SHIFTS), 20
    x = torch.tensor(SHIFTS, device="cuda").to(dtype)[:, None].expand(-1, vocab).contiguous()
    c = torch.full((beams,), -0.375, device="cuda")
    got = _select(x, c, beams, width)
    check(got, reference(x, c, beams, width))
    assert got.tokens.tolist() == [list(range(width))] and not got.parents.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_shifted_rows_tie(dtype):
    """Rows of four values, each beam's the first's and a constant, exactly."""
    beams, width, vocab = len(SHIFTS), 24, 30001
    base = torch.tensor([0.0, -0.5, -1.25, -7.0], device="cuda")
    row = base[torch.arange(vocab, device="cuda") * 7 % 11 % 4]
    row[::1009] = 0.25
    x = row + torch.tensor([4.0, -3.0, 0.0, 2.5, -2.0, 1.0, 6.0, -8.0], device="cuda")[:, None]
    x = x.to(dtype)
    c = torch.full((beams,), -2.0, device="cuda")
    check(_select(x, c, beams, width), reference(x, c, beams, width))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [3001, 151936])
def test_order_of_rows_of_few_values(vocab, dtype):
    """Two beams of few distinct logits, with scores that make their best nearly the same: up
    to half a step of fp32 apart.  The sums' terms are good to 8e-13 and the log's correction
    to as much, of either beam: pairs nearer than 1e-11 are moved apart by a step."""
    rng = np.random.default_rng([vocab, len(str(dtype))])
    seqs, beams = 48, 2
    x = torch.empty((seqs * beams, vocab), dtype=dtype)
    for r in range(seqs * beams):
        values = torch.from_numpy(rng.uniform(-6, 9, 3).astype(np.float32)).to(dtype)
        x[r] = values[torch.from_numpy(rng.choice(3, vocab, p=[0.05, 0.55, 0.4]))]
    d = x.double().numpy()
    best = d.max(1) - (np.log(np.exp(d - d.max(1, keepdims=True)).sum(1)) + d.max(1))
    c = np.empty(seqs * beams, np.float32)
    for s in range(seqs):
        a, b = 2 * s, 2 * s + 1
        c[a] = 0.0
        c[b] = np.float32(best[a] - best[b])
        while abs(np.float64(c[b]) + best[b] - best[a]) < 1e-11:
            c[b] = np.nextafter(c[b], np.float32(-100))
    x, c = x.cuda(), torch.from_numpy(c).cuda()
    check(_select(x, c, beams, 5), reference(x, c, beams, 5))


def test_the_largest_vocabulary():
    """2^24 tokens, 64 beams, 64 best: the most candidates that a sequence can have.  Other
    than the reference, a row at a time (of random fp32 logits the best hardly ever tie)."""
    beams, width, vocab = 64, 64, 1 << 24
    g = torch.Generator(device="cuda").manual_seed(11)
    c = -0.01 * torch.rand(beams, generator=g, device="cuda")
    try:
        x = torch.randn((beams, vocab), generator=g, device="cuda")
    except torch.OutOfMemoryError:
        pytest.skip("needs 8 GB")
    scores, tokens = [], []
    for r in range(beams):
        row = x[r].double()
        top = row.max()
        best = torch.topk(row, width)
        scores.append(c[r].double() + (best.values - top) - torch.exp(row - top).sum().log())
        tokens.append(best.indices)
    flat = torch.stack(scores).view(-1)
    at = flat.argsort(descending=True, stable=True)[:width]
    assert (flat[at].diff() < -1e-11).all()
    got = _select(x, c, beams, width)
    check(got, (at[None].cpu().numpy() // width, torch.stack(tokens).view(-1)[at][None].cpu().numpy(),
                flat[at][None].cpu().numpy()))
