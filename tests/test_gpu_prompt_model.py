"""Prompts through the model and the backend: DecodeModel.prefill and the per-layer
seam over packed rows against the oracle decoder, the attention backend's packed
and shared-prefix forms, and a server's run of tables, KV writes, prompt chunks,
shared-prefix decode, drafts and releases against float64 attention."""
import math

import numpy as np
import pytest
import torch

from oracle import model as omodel
from oracle import q4_0 as oq
from oracle.bf16 import bf16_bits_to_f32, round_bf16

from _rows import assert_rows, attend64, prefix64, prompt64
from _util import assert_close_rel, f32_of, pkg

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _ops():
    return pkg("native.torch_ops")


def _cfg(activation="swiglu"):
    return pkg("integration.model").DecoderConfig(
        hidden=256, n_layers=2, n_q=8, n_kv=2, head_dim=128, intermediate=512, vocab=1000,
        block_size=32, activation=activation)


def _model(dev, seed, batch=1, activation="swiglu", max_len=160, **kw):
    return pkg("integration.model").DecodeModel(_cfg(activation), dev, seed=seed, max_len=max_len,
                                                batch=batch, **kw)


def _prompts(seed, lens):
    g = np.random.default_rng(seed)
    return [g.integers(0, 1000, n) for n in lens]


def _same_greedy(gid, ol, gl, what):
    """Logits within the decode tests' bar of the oracle, the token its argmax or
    a near-tie."""
    assert_close_rel(gl, ol, rtol=2e-2, atol_frac=2e-2, what=what)
    if gid != omodel.bf16_argmax(ol):
        assert omodel.top2_margin(ol)[1] < omodel.NEAR_TIE_REL, what


def _rounded_gemv(x_f32, blocks, n, k):
    """The oracle's product over the weights' bf16 roundings, which a linear of more
    than 16 rows multiplies (smx_q4_0_gemm_rows, and the dequantised product)."""
    w = bf16_bits_to_f32(oq.c_dequant_bf16_bits(blocks, n, k)).reshape(n, k)
    return round_bf16((w.astype(np.float64) @ round_bf16(x_f32).astype(np.float64)).astype(
        np.float32))


def _pass_rows(lens, chunk):
    """For each token of each prompt the rows of the pass that takes it in."""
    done, rows = [0] * len(lens), [[] for _ in lens]
    while done != lens:
        n, room = [], chunk
        for length, at in zip(lens, done):
            n.append(min(length - at, room))
            room -= n[-1]
        for r, k in enumerate(n):
            rows[r] += [sum(n)] * k
        done = [a + b for a, b in zip(done, n)]
    return rows


@pytest.mark.parametrize("activation", ["swiglu", "gelu"])
@pytest.mark.parametrize("lens,chunk", [([1], 8192), ([2], 8192), ([40], 8192), ([100], 8192),
                                        ([100], 33), ([70], 1), ([3, 90, 17], 8192),
                                        ([3, 90, 17], 40), ([33, 1, 64, 5, 5, 2], 8192)])
def test_prefill_then_decode_against_the_oracle(dev, lens, chunk, activation, monkeypatch):
    """prefill's logits, the cache it leaves (the steps after it read it) and the
    tokens generated from it, each step of each sequence against the oracle, which
    multiplies the same weights: their bf16 roundings in passes of more than 16
    rows, the exact ones otherwise."""
    from test_gpu_model import oracle_from
    B, steps = len(lens), 4
    model = _model(dev, 31, batch=B, activation=activation)
    prompts = _prompts(7, lens)
    logits = model.prefill([torch.from_numpy(p) for p in prompts], chunk_tokens=chunk)
    record = [f32_of(logits).reshape(B, -1)]
    for _ in range(steps):
        model.step()
        torch.cuda.synchronize()
        record.append(f32_of(model.logits).reshape(B, -1))
    tokens = model.state.tokens.cpu().numpy()
    for r, p in enumerate(prompts):
        assert np.array_equal(tokens[r, :len(p)], p)
        oracle = oracle_from(model, num_splits=1)
        for pos, t in enumerate(p):
            with monkeypatch.context() as m:
                if _pass_rows(lens, chunk)[r][pos] > 16:
                    m.setattr(omodel, "_gemv", _rounded_gemv)
                ol = oracle.step(int(t), pos)
        for i in range(steps + 1):
            what = f"sequence {r} of {lens}, token {i}"
            _same_greedy(int(tokens[r, len(p) + i]), ol, record[i][r], what)
            if i < steps:
                ol = oracle.step(int(tokens[r, len(p) + i]), len(p) + i)


def test_generate_with_prefill(dev):
    """generate(prefill=True): the prompt, then new_tokens; eager, captured and on
    the runner alike, and again after another prompt."""
    a, b, c = (_model(dev, 33, num_splits=2) for _ in range(3))
    p = torch.from_numpy(_prompts(8, [50])[0])
    want = a.generate(p, 9, prefill=True)
    assert torch.equal(want[:50].cpu(), p) and want.numel() == 59
    b.capture()
    c.record_runner()
    for _ in range(2):
        assert torch.equal(b.generate(p, 9, prefill=True), want)
        assert torch.equal(c.generate(p, 9, fences="acquire", prefill=True), want)
        b.generate(p[:7], 3, prefill=True)
        c.generate(p[:7], 3, fences="agent", prefill=True)
    m = _model(dev, 33, batch=2)
    out = m.generate([p, p[:20]], 5, prefill=True)
    assert out.shape == (2, 55) and (out[0] >= 0).all()
    assert (out[1, :25] >= 0).all() and (out[1, 25:] == -1).all()
    with pytest.raises(ValueError):
        m.prefill([p, p], chunk_tokens=0)


@pytest.mark.parametrize("activation", ["swiglu", "gelu"])
def test_layer_seam_over_packed_rows(dev, activation, monkeypatch):
    """torch.ops.smx.layer_run with a query_start_loc: the model loop over two ragged
    prompts in one pass (padded by one row) against the oracle."""
    from test_gpu_model import oracle_from
    att, lr, ops = pkg("integration.attention"), pkg("integration.layer_run"), _ops()
    pkg("integration.custom_ops").register()
    model = _model(dev, 35, batch=2, activation=activation)
    c, st = model.cfg, model.state
    lens = [37, 21]
    prompts = _prompts(9, lens)
    i32 = dict(dtype=torch.int32, device=dev)
    t = ops.request_tables(torch.tensor(lens, **i32), torch.zeros(2, **i32),
                           torch.full((2,), st.block_table.shape[1], **i32),
                           torch.full((1,), -1, **i32), torch.zeros(1, **i32), st.block_table,
                           c.block_size, max_tokens=sum(lens) + 1)
    md = att.SplitKVDecodeMetadata(block_tables=st.block_table, seq_lens=t.seq_lens,
                                   slot_mapping=t.slot_mapping, num_splits=1,
                                   query_start_loc=t.query_start_loc)
    ids = torch.from_numpy(np.concatenate(prompts + [np.zeros(1, np.int64)])).to(dev)
    lr.uninstall()
    lr.install(model)
    try:
        lr.set_attention_metadata(md)
        r = model.head.embed(ids)
        y, _ = ops.add_rmsnorm(r, None, model.layers[0].input_norm, c.eps)
        for L in model.layers:
            y, r = torch.ops.smx.layer_run(y, r, t.positions, L.name)
        with pytest.raises(ValueError, match="positions"):
            lr.layer_run(y, r, t.positions[:3], model.layers[0].name)
        with pytest.raises(ValueError, match="bf16"):
            lr.layer_run(y.float(), r, t.positions, model.layers[0].name)
    finally:
        lr.uninstall()
    # 58 rows, the head's too: the products are over the weights' bf16 roundings
    logits = f32_of(ops.q4_0_gemm_rows(y, model.head.q4_0_head, c.vocab, c.hidden))
    monkeypatch.setattr(omodel, "_gemv", _rounded_gemv)
    for s, p in enumerate(prompts):
        oracle = oracle_from(model, num_splits=1)
        for pos, tok in enumerate(p):
            ol = oracle.step(int(tok), pos)
            assert_close_rel(logits[int(sum(lens[:s])) + pos], ol, rtol=2e-2, atol_frac=2e-2,
                             what=f"prompt {s} at {pos}")


def _backend_case(dev, seed, n, ctx):
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(n, ctx)]
    per = -(-max(lens) // 32)
    blocks = len(n) * per + 1
    cache = torch.randn((2, blocks, 32, 2, 128), generator=g).to(BF16)
    table = torch.randperm(blocks, generator=g)[:len(n) * per].to(torch.int32).view(-1, per)
    rows = sum(n)
    q = torch.randn((rows, 8 * 128), generator=g).to(BF16)
    k, v = (torch.randn((rows, 2 * 128), generator=g).to(BF16) for _ in range(2))
    start = np.cumsum([0] + n)
    slots = torch.tensor([int(table[r, t // 32]) * 32 + t % 32 for r in range(len(n))
                          for t in range(ctx[r], lens[r])])
    return q, k, v, cache, table, torch.tensor(start, dtype=torch.int32), lens, slots


def test_backend_forward_of_packed_rows(dev):
    att = pkg("integration.attention")
    q, k, v, cache, table, start, lens, slots = _backend_case(dev, 41, [20, 1, 7], [0, 60, 33])
    md = att.SplitKVDecodeMetadata(
        block_tables=table.to(dev), seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
        slot_mapping=slots.to(dev), num_splits=1, query_start_loc=start.to(dev))
    impl = att.SplitKVDecodeImpl(8, 128, 0.09, 2)
    kv = cache.to(dev)
    got = impl.forward(None, q.to(dev), k.to(dev), v.to(dev), kv, md)
    out = torch.empty_like(got)
    again = impl.forward(None, q.to(dev), k.to(dev), v.to(dev), kv, md, output=out)
    assert again.data_ptr() == out.data_ptr() and torch.equal(again, got)
    host = kv.cpu()
    flat = host.view(2, -1, 2, 128)
    assert torch.equal(flat[0][slots], k.view(-1, 2, 128))  # the rows' K and V were written
    assert torch.equal(flat[1][slots], v.view(-1, 2, 128))
    ref, mag, _ = prompt64(q.view(-1, 8, 128), host[0], host[1], table, start, lens, 0.09)
    assert_rows(got.view(-1, 8, 128), ref, mag, "packed rows")


def test_backend_forward_under_a_shared_prefix(dev):
    att = pkg("integration.attention")
    q, k, v, cache, table, _, lens, slots = _backend_case(dev, 43, [1] * 5, [64, 70, 99, 64, 80])
    table[:, :2] = table[0, :2]  # the first 64 tokens are one sequence's pages
    slots = torch.tensor([int(table[r, (L - 1) // 32]) * 32 + (L - 1) % 32
                          for r, L in enumerate(lens)])
    md = att.SplitKVDecodeMetadata(
        block_tables=table.to(dev), seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
        slot_mapping=slots.to(dev), num_splits=1, prefix_table=table[0, :2].to(dev),
        prefix_len=torch.tensor([64], dtype=torch.int32, device=dev))
    impl = att.SplitKVDecodeImpl(8, 128, 0.09, 2)
    kv = cache.to(dev)
    got = impl.forward(None, q.to(dev), k.to(dev), v.to(dev), kv, md)
    host = kv.cpu()
    ref, mag = prefix64(q.view(-1, 8, 128), host[0], host[1], table[0, :2], 64, table, lens, 0.09)
    assert_rows(got.view(-1, 8, 128), ref, mag, "shared prefix")
    md.query_start_loc = torch.zeros(6, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="do not go together"):
        impl.forward(None, q.to(dev), k.to(dev), v.to(dev), kv, md)


def test_custom_ops(dev):
    """The torch.ops forms: the wrappers' bits, zeros in rows of no sequence, and
    shapes under a fake mode."""
    pkg("integration.custom_ops").register()
    ops = _ops()
    q, _, _, cache, table, start, lens, _ = _backend_case(dev, 45, [9, 3], [0, 40])
    q = torch.cat((q.view(-1, 8, 128), q.view(-1, 8, 128)[:2])).to(dev)
    a = [cache[0].to(dev), cache[1].to(dev), table.to(dev)]
    start, lens = start.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    got = torch.ops.smx.prompt_attention(q, *a, start, lens, 0.1)
    assert torch.equal(got[:12], ops.prompt_attention(q, *a, start, lens, 0.1)[:12])
    assert (got[12:] == 0).all()
    plen = torch.tensor([32], dtype=torch.int32, device=dev)
    args = (q[:2].contiguous(), a[0], a[1], a[2][1, :1].contiguous(), plen, a[2], lens, 0.1)
    assert torch.equal(torch.ops.smx.shared_prefix_attention(*args),
                       ops.shared_prefix_attention(*args))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        f = [mode.from_tensor(x) for x in (q, *a, start, lens)]
        assert torch.ops.smx.prompt_attention(*f, 0.1).shape == q.shape


def test_on_the_step_runner(dev):
    """The three operators recorded once and replayed as packets: the eager bits."""
    ops, runner = _ops(), pkg("native.runner")
    q, _, _, cache, table, start, lens, _ = _backend_case(dev, 47, [4, 3], [1000, 1500])
    q = q.view(-1, 8, 128).to(dev)
    kc, vc, t = cache[0].to(dev), cache[1].to(dev), table.to(dev)
    start, lens = start.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    plen = torch.tensor([700], dtype=torch.int32, device=dev)
    ptable = t[0].contiguous()
    ws = ops.prompt_attention_workspace(q, kc, t)
    q2 = q[:2].contiguous()
    ws2 = ops.shared_prefix_attention_workspace(q2, kc, ptable, t)
    out, out2 = torch.empty_like(q), torch.empty_like(q2)
    i32 = dict(dtype=torch.int32, device=dev)
    query, context, held = torch.tensor([300, 1], **i32), torch.tensor([5, 31], **i32), \
        torch.tensor([1, 1], **i32)
    free, count, bt = torch.arange(50, **i32), torch.tensor([50], **i32), torch.full((2, 12), -1,
                                                                                     **i32)
    tabs = ops.request_tables_out(held, 5000)

    def run():
        ops.request_tables(query, context, held, free, count, bt, 32, out=tabs)
        ops.prompt_attention(q, kc, vc, t, start, lens, 0.1, workspace=ws, out=out)
        ops.shared_prefix_attention(q2, kc, vc, ptable, plen, t, lens, 0.1, workspace=ws2,
                                    out=out2)

    run()
    torch.cuda.synchronize()
    want = [x.clone() for x in (out, out2, bt, tabs.slot_mapping, tabs.positions)]
    with runner.StepRunner() as r:
        r.record(run)
        for fences in ("agent", "acquire"):
            for x in (out, out2, bt, tabs.slot_mapping, tabs.positions):
                x.fill_(-1)
            r.run(3, fences=fences)
            torch.cuda.synchronize()
            for x, w in zip((out, out2, bt, tabs.slot_mapping, tabs.positions), want):
                assert torch.equal(x, w), fences


def test_a_servers_run(dev):
    """Tables, KV writes and both attentions as a server uses them: requests come in
    under a shared system prompt, prompts are taken in by chunks, decode runs
    under the prefix, drafts are verified and some taken back, requests end and
    others take their pages.  Every attention output against float64 attention
    over the tokens' K and V as they were made."""
    ops, tables = _ops(), pkg("integration.block_table")
    S, bs, hd, n_q, n_kv, width, prefix = 4, 32, 128, 8, 2, 10, 70
    scale = 1 / math.sqrt(hd)
    g = torch.Generator().manual_seed(5)
    T = tables.DeviceBlockTables(60, bs, S, width, 512, dev)
    kc = torch.full((60, bs, n_kv, hd), math.nan, dtype=BF16, device=dev)  # never written: NaN
    vc = torch.full_like(kc, math.nan)
    kept = [[torch.zeros((0, n_kv, hd), dtype=BF16)] * 2 for _ in range(S)]  # what each holds
    i32 = dict(dtype=torch.int32, device=dev)

    def rows(n):
        return torch.randn((n, n_kv, hd), generator=g).to(BF16)

    def pass_of(n, new_kv, shared=0):
        """One step: n[r] more tokens with K and V new_kv[r]."""
        t = T.step(torch.tensor(n, **i32))
        total = sum(n)
        for r in range(S):
            kept[r] = [torch.cat((a, b)) for a, b in zip(kept[r], new_kv[r])]
        ops.reshape_and_cache(torch.cat([x[0] for x in new_kv]).to(dev),
                              torch.cat([x[1] for x in new_kv]).to(dev), kc, vc,
                              t.slot_mapping[:total])
        q = torch.randn((total, n_q, hd), generator=g).to(BF16)
        if shared:
            got = ops.shared_prefix_attention(q.to(dev), kc, vc, T.block_table[0], shared_len,
                                              T.block_table, t.seq_lens, scale)
        else:
            out = torch.zeros((total + 3, n_q, hd), dtype=BF16, device=dev)
            qp = torch.cat((q, q[:1].expand(3, -1, -1))).to(dev)
            got = ops.prompt_attention(qp, kc, vc, T.block_table, t.query_start_loc, t.seq_lens,
                                       scale, out=out)
            assert (got[total:] == 0).all()
        at = 0
        for r in range(S):
            if not n[r]:
                continue
            L = kept[r][0].shape[0]
            seen = torch.arange(L)[None] <= torch.arange(L - n[r], L)[:, None]
            ref, mag = attend64(q[at:at + n[r]].double(), kept[r][0].double(),
                                kept[r][1].double(), scale, seen)
            assert_rows(got[at:at + n[r]], ref, mag, f"request {r}, {n}")
            at += n[r]

    shared_len = torch.tensor([prefix], **i32)
    system = [rows(prefix), rows(prefix)]
    # the system prompt in two chunks, every request with pages of its own
    pass_of([40] * S, [[x[:40] for x in system]] * S)
    pass_of([30] * S, [[x[40:] for x in system]] * S)
    pass_of([5, 90, 1, 33], [[rows(k), rows(k)] for k in (5, 90, 1, 33)])
    for _ in range(3):  # decode under the prefix
        pass_of([1] * S, [[rows(1), rows(1)] for _ in range(S)], shared=1)
    for accepted in ([3, 0, 4, 2], [0, 1, 1, 4]):  # drafts: 4 a request, some taken back
        before = [x[0].shape[0] for x in kept]
        pass_of([4] * S, [[rows(4), rows(4)] for _ in range(S)])
        T.keep(torch.tensor([a + b for a, b in zip(before, accepted)], **i32))
        kept = [[x[:a + b] for x in kv] for kv, a, b in zip(kept, before, accepted)]
    T.keep(torch.tensor([kept[0][0].shape[0], 0, kept[2][0].shape[0], 0], **i32))  # two end
    for r in (1, 3):
        kept[r] = [x[:0] for x in kept[r]]
    assert T.lens.tolist() == [x[0].shape[0] for x in kept]
    pass_of([1, 60, 1, 0], [[rows(k), rows(k)] for k in (1, 60, 1, 0)])
    held = [p for row, k in zip(T.block_table.tolist(), T.num_pages.tolist()) for p in row[:k]]
    free = T.free_pages.tolist()[:int(T.free_count)]
    assert sorted(held + free) == list(range(60))
