"""Beam search's selection: zeros of either sign are equal logits, wherever they stand."""
import pytest
import torch

from _util import pkg
from test_gpu_beam_select import check, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [1, 2, 3, 7])
@pytest.mark.parametrize("rest", [-1.0, -100.0])
def test_zeros_of_both_signs_apart(rest, width, dtype):
    """Few zeros in loads of their own among negative logits: those of a negative sign tie with
    the others, and the lowest tokens come first.  Two beams of the same row and score, so
    that the order of the beams counts too."""
    print(rest, width, dtype, flush=True)
    beams, vocab = 2, 40000
    for minus, plus in (([0], [64]), ([5, 300], [2, 9000]), ([17, 39999], [18000, 20000]),
                        ([1, 8, 16, 24], [32]), ([70], [0, 8, 16]), ([3, 4, 700], [])):
        row = torch.full((vocab,), rest, device="cuda")
        row[minus], row[plus] = -0.0, 0.0
        x = row.to(dtype).expand(beams, vocab).contiguous()
        c = torch.zeros(beams, device="cuda")
        check(pkg("native.torch_ops").beam_select(x, c, beams, width),
              reference(x, c, beams, width), f"{minus} {plus}")
