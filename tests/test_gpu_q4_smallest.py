"""The smallest blocks that a KV cache in 4 bits holds: up to a largest magnitude of 2^-22 their
scale is 0 (2^-25 is half of fp16's least) and their codes 8, above it they have a value."""
import pytest
import torch

from _util import pkg
from oracle import q4_kv

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_scales_on_both_sides_of_2_22():
    ops = pkg("native.torch_ops")
    tops = torch.tensor([2.0 ** -22, 2.0 ** -22 * (1 + 2.0 ** -7), 2.0 ** -23, 2.0 ** -21, 2.0 ** -133])
    tops = torch.cat((tops, -tops))
    key = tops[:, None, None] * torch.linspace(1, -1, 64)
    key = key.to(BF16)
    key[..., 32] = tops[:, None].to(BF16)
    cache = ops.q4_kv_cache(1, 32, 1, 64, "cuda")
    slots = torch.arange(10, device="cuda")
    ops.reshape_and_cache_q4(key.cuda(), key.cuda(), cache, slots)
    codes, d = q4_kv.quantise(key.double().numpy())
    assert [bool(x) for x in d[:, 0].any(-1)] == [False, True, False, True, False] * 2
    got_k, got_v = ops.q4_kv_read(cache, slots)
    want = torch.from_numpy(q4_kv.values(codes, d)).float()
    assert torch.equal(got_k.cpu(), want) and torch.equal(got_v.cpu(), want)
    raw = cache.scales[0, 0, 0, :10].cpu()
    assert torch.equal(raw, torch.from_numpy(d[:, 0]))
