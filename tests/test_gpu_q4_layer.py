"""The decoder layer over a cache in 4 bits (layer_run, prompt_layer): packed prompts and
then decode steps, against its operators one by one and against bf16 writes quantised."""
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _model(batch):
    m = pkg("integration.model")
    cfg = m.DecoderConfig(n_layers=2, hidden=512, n_q=8, n_kv=2, head_dim=128, intermediate=1024,
                          vocab=1000, block_size=32)
    return m.DecodeModel(cfg, "cuda", seed=3, max_len=256, num_splits=2, batch=batch)


def test_prompts_and_decode_steps():
    ops, att, lr = pkg("native.torch_ops"), pkg("integration.attention"), pkg("integration.layer_run")
    tab = pkg("integration.block_table")
    model = _model(2)
    c = model.cfg
    for L in model.layers:
        L.kv_cache = att.SplitKVDecodeBackend.get_q4_kv_cache(16, c.block_size, c.n_kv, c.head_dim,
                                                              "cuda")
    kept = [L.kv_cache for L in model.layers]
    tables = tab.DeviceBlockTables(16, c.block_size, 2, 8, 80, "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    lr.uninstall()
    lr.install(model)

    def by_hand(x, res, L, nxt, positions, t, start):
        qkv = L.qkv.quant_method.apply(L.qkv, x)
        # (into a copy, and its bf16 K and V, quantised, into another)
        cache, other = (ops.Q4KVCache(L.kv_cache.codes.clone(), L.kv_cache.scales.clone())
                        for _ in range(2))
        q = ops.qknorm_rope_kv_write_q4(qkv, L.q_norm, L.k_norm, model.cos_sin, positions,
                                        t.slot_mapping[:len(x)], cache, c.n_q, c.n_kv, c.eps)
        kv = torch.zeros((2, 16, c.block_size, c.n_kv, c.head_dim), dtype=BF16, device="cuda")
        assert torch.equal(q, ops.qknorm_rope_kv_write(
            qkv, L.q_norm, L.k_norm, model.cos_sin, positions, t.slot_mapping[:len(x)], kv[0],
            kv[1], c.n_q, c.n_kv, c.eps))
        slots = t.slot_mapping[:len(x)][t.slot_mapping[:len(x)] >= 0]
        k, v = (p.view(-1, c.n_kv, c.head_dim)[slots] for p in kv)
        ops.reshape_and_cache_q4(k, v, other, slots)
        assert torch.equal(cache.codes, other.codes) and torch.equal(cache.scales, other.scales)
        o = ops.q4_attention(q, cache, tables.block_table, t.seq_lens, model.scale,
                             query_start_loc=start, out=torch.zeros_like(q))
        o = L.o_proj.quant_method.apply(L.o_proj, o.view(len(x), -1))
        h, res = ops.add_rmsnorm(o, res, L.post_norm, c.eps)
        act = ops.silu_mul(L.gate_up.quant_method.apply(L.gate_up, h))
        y, res = ops.add_rmsnorm(L.down.quant_method.apply(L.down, act), res, nxt, c.eps)
        return y, res, cache

    try:
        for n, packed in (([45, 30], True), ([1, 1], False), ([1, 1], True), ([3, 2], True),
                          ([1, 1], False)):
            print(n, packed, flush=True)
            t = tables.step(torch.tensor(n, dtype=torch.int32, device="cuda"))
            rows = sum(n)
            start = t.query_start_loc if packed else None
            md = att.SplitKVDecodeMetadata(
                block_tables=tables.block_table, seq_lens=t.seq_lens,
                slot_mapping=t.slot_mapping[:rows], num_splits=1, query_start_loc=start)
            lr.set_attention_metadata(md)
            x = torch.randn((rows, c.hidden), generator=g, device="cuda").to(BF16)
            res = torch.randn((rows, c.hidden), generator=g, device="cuda").to(BF16)
            for i, L in enumerate(model.layers):
                nxt = model.layers[i + 1].input_norm if i + 1 < len(model.layers) \
                    else model.final_norm
                y2, r2, cache = by_hand(x, res, L, nxt, t.positions[:rows], t, start)
                x, res = lr.layer_run(x, res, t.positions[:rows], L.name)
                assert L.kv_cache is kept[i]
                assert torch.equal(x, y2) and torch.equal(res, r2)
                assert torch.equal(L.kv_cache.codes, cache.codes)
                assert torch.equal(L.kv_cache.scales, cache.scales)
                assert torch.isfinite(x).all()
        with pytest.raises(ValueError, match="4 bits"):
            lr.layer_run(x[:1], res[:1], t.positions[:1], model.layers[0].name)
        lr.set_attention_metadata(None)
        with pytest.raises(RuntimeError, match="metadata"):
            lr.layer_run(x, res, t.positions[:2], model.layers[0].name)
    finally:
        lr.uninstall()
