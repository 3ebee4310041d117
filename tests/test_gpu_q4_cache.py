"""Writes to and reads from a KV cache held in 4 bits (torch_ops.reshape_and_cache_q4,
qknorm_rope_kv_write_q4, q4_kv_read) against a float64 restatement: codes, scales and
values are equal, bit for bit."""
import numpy as np
import pytest
import torch

from _util import bf16_dev, pkg
from oracle import q4_kv
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ops():
    return pkg("native.torch_ops")


def _bits(rng, shape, kind):
    x = rng.standard_normal(shape).astype(np.float32)
    if kind == "channels":  # some channels a thousand times the others
        x *= np.exp(2 * rng.standard_normal(shape[-1])).astype(np.float32)
    elif kind == "borders":  # multiples of an eighth of a power of two: quotients on borders
        x = (rng.integers(-16, 17, shape) / 16).astype(np.float32)
        x[..., rng.integers(0, shape[-1])] = -1.0
    elif kind == "tiny":
        x *= np.float32(2.0) ** rng.integers(-40, -10, (*shape[:-1], 1))
    elif kind == "huge":
        x *= np.float32(2.0) ** rng.integers(10, 100, (*shape[:-1], 1))
    elif kind == "ties":  # the largest magnitude several times, of both signs
        x = rng.choice(np.array([-2.0, 2.0, 0.5, 0.0, -0.0], np.float32), shape)
    elif kind == "odd":
        flat = x.reshape(-1)
        for v in (np.inf, -np.inf, np.nan, 0.0):
            flat[rng.integers(0, flat.size, max(1, flat.size // 300))] = v
        x.reshape(-1, 32)[::7] = 0.0
    return f32_to_bf16_bits(x)


@pytest.mark.parametrize("kind", ["plain", "channels", "borders", "tiny", "huge", "ties", "odd"])
@pytest.mark.parametrize("tokens,n_kv,hd,bs", [(1, 1, 64, 32), (1, 8, 128, 128), (37, 3, 128, 32),
                                               (130, 2, 64, 64), (5, 16, 128, 4096)])
def test_writes_and_reads(kind, tokens, n_kv, hd, bs):
    print(kind, tokens, n_kv, hd, bs, flush=True)
    ops = _ops()
    rng = np.random.default_rng([tokens, n_kv, hd, bs, len(kind)])
    blocks = -(-tokens // bs) + 2
    cache = ops.q4_kv_cache(blocks, bs, n_kv, hd, "cuda")
    cache.codes.fill_(0x5a)
    cache.scales.fill_(3.0)
    kv = [_bits(rng, (tokens, n_kv, hd), kind) for _ in range(2)]
    slots = rng.permutation(blocks * bs)[:tokens]
    skipped = tokens // 3
    slots[:skipped:2] = -1
    slots[1:skipped:2] = blocks * bs + 5
    dev = [bf16_dev(x, "cuda") for x in kv]
    s = torch.tensor(slots, device="cuda")
    ops.reshape_and_cache_q4(*dev, cache, s)
    codes, scales = cache.codes.cpu().numpy(), cache.scales.cpu().numpy()
    want_c = np.full(codes.shape, 0x5a, np.uint8)
    want_s = np.full(scales.shape, 3.0, np.float16)
    read = ops.q4_kv_read(cache, s)
    for i in range(2):
        c, d = q4_kv.quantise(bf16_bits_to_f32(kv[i]))
        packed = q4_kv.pack(c, i == 0)
        val = q4_kv.values(c, d)
        for t, slot in enumerate(slots):
            if 0 <= slot < blocks * bs:
                want_c[i, slot // bs, :, slot % bs] = packed[t]
                want_s[i, slot // bs, :, slot % bs] = d[t]
            else:
                val[t] = 0.0
        np.testing.assert_array_equal(read[i].cpu().numpy(), val.astype(np.float32))
    np.testing.assert_array_equal(scales, want_s)
    np.testing.assert_array_equal(codes, want_c)


def test_codes_are_nearest_and_errors_are_half_a_step():
    """|value - x| <= |d| / 2 but for x beyond the codes' end (+8 d, held as 7 d)."""
    rng = np.random.default_rng(5)
    x = bf16_bits_to_f32(_bits(rng, (64, 4, 128), "channels")).astype(np.float64)
    c, d = q4_kv.quantise(x)
    step = np.repeat(np.abs(d.astype(np.float64)), 32, -1)
    err = np.abs(q4_kv.values(c, d) - x)
    assert (err <= np.where(c == 15, step, step / 2 * (1 + 2.0 ** -9))).all()


def test_strided_tokens():
    """K and V taken out of the QKV rows as they are."""
    ops = _ops()
    rng = np.random.default_rng(6)
    n_q, n_kv, hd, t = 8, 2, 128, 19
    qkv = bf16_dev(_bits(rng, (t, (n_q + 2 * n_kv) * hd), "plain"), "cuda").view(t, -1, hd)
    s = torch.arange(t, device="cuda")
    caches = [ops.q4_kv_cache(2, 32, n_kv, hd, "cuda") for _ in range(2)]
    k, v = qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:]
    ops.reshape_and_cache_q4(k, v, caches[0], s)
    ops.reshape_and_cache_q4(k.contiguous(), v.contiguous(), caches[1], s)
    assert torch.equal(caches[0].codes, caches[1].codes)
    assert torch.equal(caches[0].scales, caches[1].scales)
    assert caches[0].codes.any()


@pytest.mark.parametrize("tokens,n_q,n_kv,bs", [(1, 32, 8, 128), (3, 4, 1, 32), (70, 6, 2, 64)])
def test_norm_rope_and_write(tokens, n_q, n_kv, bs):
    """qknorm_rope_kv_write_q4 is qknorm_rope_kv_write and a write of what that kept.
    (Both kernels of the latter round alike.)"""
    print(tokens, n_q, n_kv, bs, flush=True)
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF16)  # noqa: E731
    qkv, qg, kg, cs = rand(tokens, (n_q + 2 * n_kv) * 128), rand(128), rand(128), rand(500, 128)
    pos = torch.randint(-2, 600, (tokens,), generator=g, device="cuda")
    blocks = -(-tokens // bs) + 1
    slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[1] = -1
    kc, vc = (torch.zeros((blocks, bs, n_kv, 128), dtype=BF16, device="cuda") for _ in range(2))
    q = ops.qknorm_rope_kv_write(qkv, qg, kg, cs, pos, slots, kc, vc, n_q, n_kv, 1e-6)
    cache, want = (ops.q4_kv_cache(blocks, bs, n_kv, 128, "cuda") for _ in range(2))
    q4 = ops.qknorm_rope_kv_write_q4(qkv, qg, kg, cs, pos, slots, cache, n_q, n_kv, 1e-6)
    assert torch.equal(q.view(torch.int16), q4.view(torch.int16))
    at = slots.clamp(min=0)
    ops.reshape_and_cache_q4(kc.view(-1, n_kv, 128)[at], vc.view(-1, n_kv, 128)[at], want, slots)
    assert torch.equal(cache.codes, want.codes) and torch.equal(cache.scales, want.scales)


def test_refusals():
    ops = _ops()
    cache = ops.q4_kv_cache(4, 32, 2, 64, "cuda")
    x = torch.zeros((3, 2, 64), dtype=BF16, device="cuda")
    s = torch.zeros(3, dtype=torch.int64, device="cuda")
    bad = [lambda: ops.reshape_and_cache_q4(x[:2], x, cache, s),
           lambda: ops.reshape_and_cache_q4(x.float(), x, cache, s),
           lambda: ops.reshape_and_cache_q4(x, x.cpu(), cache, s),
           lambda: ops.reshape_and_cache_q4(x, x, cache, s.int()),
           lambda: ops.reshape_and_cache_q4(x, x, (cache.codes, cache.scales), s),
           lambda: ops.reshape_and_cache_q4(x.transpose(0, 1).contiguous().transpose(0, 1), x,
                                            cache, s),
           lambda: ops.reshape_and_cache_q4(x[:1].expand(3, 2, 64), x, cache, s),
           lambda: ops.q4_kv_read(cache, s.int()),
           lambda: ops.q4_kv_read(cache, s, out=(x.float(), x.float()[:2])),
           lambda: ops.q4_kv_cache(4, 48, 2, 64, "cuda"),
           lambda: ops.q4_kv_cache(4, 32, 2, 96, "cuda"),
           lambda: ops.Q4KVCache(cache.codes, cache.scales[..., :1].contiguous()),
           lambda: ops.Q4KVCache(cache.codes[:1], cache.scales),
           lambda: ops.Q4KVCache(cache.codes, cache.scales.float())]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
    ops.reshape_and_cache_q4(x[:0], x[:0], cache, s[:0])  # no tokens: nothing to do
    assert ops.q4_kv_read(cache, s[:0])[0].shape == (0, 2, 64)
