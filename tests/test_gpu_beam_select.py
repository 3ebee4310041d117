"""Beam search's selection (torch_ops.beam_select) against float64 log-softmaxes and a
sort: rows and tokens equal, scores to half a step of fp32."""
import math

import numpy as np
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ops():
    return pkg("native.torch_ops")


def reference(logits, scores, beams, width, done=None, pad_id=0):
    """(parents, tokens, float64 scores), by the definition."""
    x = logits.double().cpu().numpy()
    c = scores.double().cpu().numpy()
    rows, vocab = x.shape
    x = np.where(np.isnan(x), -np.inf, x)
    total = np.full((rows, vocab), -np.inf)
    for r in range(rows):
        if not c[r] > -np.inf:
            continue
        if done is not None and bool(done[r]):
            total[r, pad_id] = c[r]
            continue
        top = x[r].max()
        if top == -np.inf:
            continue
        rel = np.where(x[r] == top, 0.0, x[r] - (top if np.isfinite(top) else 0.0))
        if top == np.inf:
            rel = np.where(x[r] == top, 0.0, -np.inf)
        total[r] = c[r] + (rel - np.log(np.exp(rel).sum()))
    parents, tokens, best = [], [], []
    for s in range(rows // beams):
        flat = total[s * beams:(s + 1) * beams].reshape(-1)
        order = np.argsort(-flat, kind="stable")[:width]
        order = order[flat[order] > -np.inf]
        none = [-1] * (width - len(order))
        parents.append([s * beams + int(i) // vocab for i in order] + none)
        tokens.append([int(i) % vocab for i in order] + none)
        best.append([flat[i] for i in order] + [-np.inf] * len(none))
    return np.array(parents), np.array(tokens), np.array(best)


def check(got, ref, what=""):
    parents, tokens, best = ref
    np.testing.assert_array_equal(got.parents.cpu().numpy(), parents, err_msg=f"{what} parents")
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens, err_msg=f"{what} tokens")
    s = got.scores.double().cpu().numpy()
    np.testing.assert_array_equal(np.isinf(s), np.isinf(best))
    fin = np.isfinite(best)
    # rounded to fp32 once; 4e-11 of the exponentials is next to nothing
    assert (np.abs(s[fin] - best[fin]) <= 2.0 ** -24 * np.abs(best[fin]) + 1e-9).all(), what


def _inputs(seed, seqs, beams, vocab, dtype=BF16, std=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((seqs * beams, vocab), generator=g, device="cuda") * std).to(dtype)
    return x, -20 * torch.rand(seqs * beams, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("seqs,beams,width,vocab", [
    (1, 1, 1, 1), (1, 1, 4, 3), (2, 3, 5, 7), (1, 4, 8, 151936), (3, 4, 4, 4095),
    (2, 5, 10, 4097), (1, 64, 64, 1000), (1, 2, 64, 50257), (7, 8, 16, 16385),
    (40, 16, 16, 32003), (65, 8, 3, 2049)])
def test_matches_float64(seqs, beams, width, vocab, dtype):
    print(seqs, beams, width, vocab, dtype, flush=True)
    x, c = _inputs(1, seqs, beams, vocab, dtype)
    check(_ops().beam_select(x, c, beams, width), reference(x, c, beams, width))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows", [4, 520])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "zeros of both signs"])
def test_ties_and_sorted_rows(kind, rows, dtype):
    """Equal scores go to the lowest beam and token; rows in order make every bound loose."""
    beams, width, vocab = 4, 9, 20011
    print(kind, rows, dtype, flush=True)
    at = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"equal": at * 0 + 1.5, "rising": at / 512 - 10, "falling": 10 - at / 512,
           "two values": (at % 3 == 1).float(),
           "zeros of both signs": torch.where(at % 2 == 0, -0.0, 0.0)}[kind]
    x = row.to(dtype).expand(rows, vocab).contiguous()
    # pairs of beams with the same score: equal all through
    c = (torch.arange(rows, device="cuda") // 2).float() * -0.25
    check(_ops().beam_select(x, c, beams, width), reference(x, c, beams, width), kind)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_masks_infinities_and_nan(dtype):
    """Rows that nothing is left of, one or few tokens, values of the type's lowest, NaN and
    infinities, beams without a score."""
    beams, width, vocab = 8, 16, 40000
    x, c = _inputs(2, 2, beams, vocab, dtype)
    low = torch.finfo(dtype).min
    x[0] = -torch.inf
    x[1] = low
    x[2, 5:] = -torch.inf
    x[3, ::2] = torch.nan
    x[4, 39999] = torch.inf
    x[5, 100:200] = torch.inf
    x[6] = torch.nan
    x[7, 1:] = low
    c[9] = -torch.inf
    c[10] = torch.nan
    x[11, :39990] = -torch.inf
    got, ref = _ops().beam_select(x, c, beams, width), reference(x, c, beams, width)
    check(got, ref)
    # nothing at all, and fewer than the width
    x[:beams] = -torch.inf
    x[beams:] = -torch.inf
    x[beams + 4, [7, 39000]] = torch.tensor([1.0, 2.0], dtype=dtype, device="cuda")
    got, ref = _ops().beam_select(x, c, beams, width), reference(x, c, beams, width)
    check(got, ref)
    assert (got.tokens[0] == -1).all() and (got.tokens[1] >= 0).sum() == 2


@pytest.mark.parametrize("pad_id", [0, 777])
def test_done_beams(pad_id):
    """A beam that is done offers pad_id at its own score; all of them done."""
    beams, width, vocab = 4, 6, 5000
    x, c = _inputs(3, 3, beams, vocab)
    done = torch.tensor([0, 1, 0, 0, 1, 1, 1, 1, 0, 0, 0, 1], dtype=torch.bool, device="cuda")
    c[1], c[4], c[5] = -0.5, -1.0, -1.0
    c[11] = -torch.inf
    x[1] = torch.nan  # (what a done beam's row holds does not matter)
    check(_ops().beam_select(x, c, beams, width, done=done, pad_id=pad_id),
          reference(x, c, beams, width, done, pad_id))


def test_close_beams():
    """Beams whose sums differ by less than fp32 holds: the order is that of 64 bits."""
    beams, vocab = 2, 30000
    x = torch.randn((2, vocab), device="cuda").to(BF16).float()
    x[1] = x[0]
    x[:, 17] = 9.0
    x[1, 5] = x[1, 5] + 1e-2  # sum larger by about 1e-7 of itself: its best is below
    x[:, 5] -= 12
    check(_ops().beam_select(x, torch.zeros(2, device="cuda"), beams, 8),
          reference(x, torch.zeros(2), beams, 8))


def test_strided_rows_and_alignment():
    """Rows of a wider head's output, any start."""
    for dtype in (BF16, torch.float32):
        for shift in (0, 1, 3):
            x, c = _inputs(4, 2, 3, 10007, dtype)
            part = x[:, shift:shift + 9001]
            check(_ops().beam_select(part, c, 3, 7), reference(part, c, 3, 7), f"{dtype} {shift}")


def test_in_place_scores_other_stream_and_capture():
    """A search's steps in one graph: scores updated in place, every replay on other logits,
    a poisoned workspace, work on another stream."""
    ops = _ops()
    beams = 4
    x, c = _inputs(5, 3, beams, 33000)
    ws = ops.beam_select_workspace(x, beams, beams)
    out = ops.beam_select_out(3, beams, "cuda")
    out = ops.BeamSelection(out.parents, out.tokens, c.view(3, beams))
    call = lambda: ops.beam_select(x, c, beams, beams, workspace=ws, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        y, d = _inputs(6 + i, 3, beams, 33000)
        x.copy_(y)
        c.copy_(d)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        check(out, reference(y, d, beams, beams), f"replay {i}")
        assert torch.equal(out.scores.view(-1), c)


def test_refusals():
    ops = _ops()
    x, c = _inputs(7, 1, 2, 100)
    f = lambda **k: ops.beam_select(**{**dict(logits=x, scores=c, beams=2, width=3), **k})  # noqa: E731
    f()
    out = ops.beam_select_out(1, 3, "cuda")
    bad = [dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.t()),
           dict(scores=c.double()), dict(scores=c[:1]), dict(scores=c.cpu()), dict(beams=0),
           dict(beams=3), dict(beams=65), dict(width=0), dict(width=65), dict(pad_id=100),
           dict(pad_id=-1), dict(done=torch.zeros(2, device="cuda")),
           dict(done=torch.zeros(1, dtype=torch.bool, device="cuda")), dict(out=(1, 2, 3)),
           dict(out=out, width=4), dict(logits=x.expand(2, 100)[:, :1].expand(2, 100)),
           dict(workspace=torch.empty(10, device="cuda"))]
    for i, change in enumerate(bad):
        with pytest.raises(ValueError):
            f(**change)
            print("not refused:", i)
    with pytest.raises(pkg("native").SmxError):
        f(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("shift,scale", [(15.0, 1.0), (16.0, 0.0), (40.0, 1.0), (-60.0, 1.0),
                                         (0.0, 10.0), (-300.0, 30.0), (1e4, 100.0), (3e38, 0.0),
                                         (-3e38, 0.0), (0.0, 1e-4)])
def test_logits_of_any_size(shift, scale, dtype):
    """Near 0, where exponentials are taken as they are, on the border, and far from it."""
    for seqs, beams, width, vocab in ((2, 3, 4, 5000), (1, 2, 16, 40001)):
        x, c = _inputs(9, seqs, beams, vocab, torch.float32, std=1.0)
        x = (x * scale + shift).to(dtype)
        x[:, ::7] = -math.inf
        check(_ops().beam_select(x, c, beams, width), reference(x, c, beams, width),
              f"{shift} {scale}")


@pytest.mark.parametrize("dtype,bits", [
    (BF16, [0x7fc0, 0x7f81, 0xffc0 - 65536, 0xff81 - 65536, 0xffff - 65536, 0x7fff]),
    (torch.float32, [0x7fc00000, 0x7f800001, 0xffc00000 - 2 ** 32, 0xff800001 - 2 ** 32, -1,
                     0x7fffffff])])
def test_every_kind_of_nan(dtype, bits):
    """Quiet and signalling, with and without a sign: never chosen, nothing in the sum."""
    x, c = _inputs(10, 2, 3, 9001, dtype)
    clean = x.clone()
    clean[:, 5::11] = -math.inf
    raw = x.view(torch.int16 if dtype is BF16 else torch.int32)
    for i, b in enumerate(bits):
        at = torch.arange(5, 9001, 11, device="cuda")[i::len(bits)]
        raw[:, at] = b
    assert x[:, 5::11].isnan().all()
    got, want = _ops().beam_select(x, c, 3, 8), _ops().beam_select(clean, c, 3, 8)
    for a, b in ((got.parents, want.parents), (got.tokens, want.tokens), (got.scores, want.scores)):
        assert torch.equal(a, b)
    check(got, reference(clean, c, 3, 8))
