"""Torch-tensor wrappers over the C ABI (the role of the reference's
TORCH_LIBRARY wrapper, src/spark_vllm_ascend/native/head/extension.cpp:6-14).

Each wrapper checks device, dtype, contiguity and element counts before the
call (raising ValueError, as TORCH_CHECK raises c10::Error), passes raw data
pointers plus the current HIP stream of the tensor's device, and returns the
output tensor.  Outputs can be passed in (``out=``) so that a captured graph
reuses fixed buffers; otherwise they are freshly allocated, as the
reference's custom ops do (src/spark_vllm_ascend/integration/head.py:8-9).
"""
from __future__ import annotations

import torch

from . import SMX_EINVAL, SmxError, call, load

BF16 = torch.bfloat16


def _stream(t: torch.Tensor) -> int:
    """The current HIP stream of the tensor's device.  (The raw getter: 0.14 us;
    torch.cuda.current_stream() builds a Stream object for its handle, 2.0 us.)"""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, numel: int | None = None,
           device: torch.device | None = None) -> None:
    # one condition for a valid tensor; what is wrong is worked out, and its
    # message formatted, only for one that is not (a call makes up to 13 checks)
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.is_contiguous()
            and (numel is None or t.numel() == numel) and (device is None or t.device == device)):
        _refuse(t, name, dtype, numel, device)


def _refuse(t, name, dtype, numel, device) -> None:
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.is_cuda, f"{name} must be on a GPU device")
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _need(t.is_contiguous(), f"{name} must be contiguous")
    if numel is not None:
        _need(t.numel() == numel, f"{name} must have {numel} elements, got {t.numel()}")
    if device is not None:
        _need(t.device == device, f"{name} must be on {device}, got {t.device}")
    raise ValueError(f"{name} is not a valid argument")


def q4_0_row_bytes(k: int) -> int:
    """Bytes of one Q4_0 row of k weights (k/32 blocks of 18 bytes)."""
    return k // 32 * 18


def q4_0_dequant_bf16(w: torch.Tensor, n: int, k: int, out: torch.Tensor | None = None) -> torch.Tensor:
    _need(k % 32 == 0 and k > 0 and n > 0, "need n > 0 and k a positive multiple of 32")
    _check(w, "w", torch.uint8, n * q4_0_row_bytes(k))
    if out is None:
        out = torch.empty((n, k), dtype=BF16, device=w.device)
    _check(out, "out", BF16, n * k, w.device)
    call("smx_q4_0_dequant_bf16", _stream(w), w.data_ptr(), out.data_ptr(), n, k)
    return out


def q4_0_gemv(x: torch.Tensor, w: torch.Tensor, n: int, k: int,
              out: torch.Tensor | None = None) -> torch.Tensor:
    _need(k % 32 == 0 and k > 0 and n > 0, "need n > 0 and k a positive multiple of 32")
    _check(x, "x", BF16, k)
    _check(w, "w", torch.uint8, n * q4_0_row_bytes(k), x.device)
    if out is None:
        out = torch.empty((1, n), dtype=BF16, device=x.device)
    _check(out, "out", BF16, n, x.device)
    call("smx_q4_0_gemv", _stream(x), x.data_ptr(), w.data_ptr(), out.data_ptr(), n, k)
    return out


GELU_LUT_ENTRIES = 4096


def gelu_table(device: torch.device | str = "cpu") -> torch.Tensor:
    """The reference's erf-GELU activation table (src/spark_vllm_ascend/
    integration/model.py:13-16): gelu(approximate='none') of the bf16 bit
    patterns 0x3b00..0x42ff, then of 0xbb00..0xc2ff, as 4096 bf16 values.
    Evaluated by torch on the CPU (the reference evaluates it on its device),
    then copied to `device`."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    full = torch.nn.functional.gelu(bits, approximate="none")
    return torch.cat((full[0x3B00:0x4300], full[0xBB00:0xC300])).contiguous().to(device)


def _lut_checked(lut: torch.Tensor, device: torch.device) -> int:
    _check(lut, "lut", BF16, GELU_LUT_ENTRIES, device)
    return lut.data_ptr()


def _gemv_gated(x, w, d, k, out, lut):
    _need(k % 32 == 0 and k > 0 and d > 0, "need d > 0 and k a positive multiple of 32")
    _check(x, "x", BF16, k)
    _check(w, "w", torch.uint8, 2 * d * q4_0_row_bytes(k), x.device)
    if out is None:
        out = torch.empty((1, d), dtype=BF16, device=x.device)
    _check(out, "out", BF16, d, x.device)
    if lut is None:
        call("smx_q4_0_gemv_swiglu", _stream(x), x.data_ptr(), w.data_ptr(), out.data_ptr(), d, k)
    else:
        call("smx_q4_0_gemv_gelu", _stream(x), x.data_ptr(), w.data_ptr(),
             _lut_checked(lut, x.device), out.data_ptr(), d, k)
    return out


def q4_0_gemv_swiglu(x: torch.Tensor, w: torch.Tensor, d: int, k: int,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    return _gemv_gated(x, w, d, k, out, None)


def q4_0_gemv_gelu(x: torch.Tensor, w: torch.Tensor, lut: torch.Tensor, d: int, k: int,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """out [1, d] = act(x W_gate^T) * (x W_up^T), act the table GELU
    (gelu_table)."""
    return _gemv_gated(x, w, d, k, out, lut)


def splitkv_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, seq_lens: torch.Tensor, num_splits: int,
                   scale: float, partial_o: torch.Tensor | None = None,
                   partial_lse: torch.Tensor | None = None):
    """Split-KV partials.  q [S, n_q, 128]; caches [blocks, bs, n_kv, 128]."""
    _need(q.dim() == 3 and k_cache.dim() == 4, "q must be [seqs, n_q, hd], caches 4-D")
    num_seqs, n_q, hd = q.shape
    num_blocks, bs, n_kv, hd2 = k_cache.shape
    _need(hd == hd2, "head_dim mismatch between q and the cache")
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    _check(q, "q", BF16)
    _check(k_cache, "k_cache", BF16, device=q.device)
    _check(v_cache, "v_cache", BF16, device=q.device)
    _check(block_table, "block_table", torch.int32, device=q.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == num_seqs, "block_table must be [seqs, max_blocks]")
    _check(seq_lens, "seq_lens", torch.int32, num_seqs, q.device)
    if partial_o is None:
        partial_o = torch.empty((num_seqs, num_splits, n_q, hd), dtype=torch.float32, device=q.device)
    if partial_lse is None:
        partial_lse = torch.empty((num_seqs, num_splits, n_q), dtype=torch.float32, device=q.device)
    _check(partial_o, "partial_o", torch.float32, num_seqs * num_splits * n_q * hd, q.device)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, q.device)
    call("smx_splitkv_decode", _stream(q), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
         block_table.data_ptr(), seq_lens.data_ptr(), partial_o.data_ptr(), partial_lse.data_ptr(),
         num_seqs, num_splits, block_table.shape[1], num_blocks, bs, n_q, n_kv, hd, float(scale))
    return partial_o, partial_lse


def splitkv_decode_merged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          block_table: torch.Tensor, seq_lens: torch.Tensor, num_splits: int,
                          scale: float, partial_o: torch.Tensor, partial_lse: torch.Tensor,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """Split-KV decode then the LSE merge, enqueued by one call; partial_o /
    partial_lse are the workspace between the two kernels."""
    _need(q.dim() == 3 and k_cache.dim() == 4, "q must be [seqs, n_q, hd], caches 4-D")
    num_seqs, n_q, hd = q.shape
    num_blocks, bs, n_kv, hd2 = k_cache.shape
    _need(hd == hd2, "head_dim mismatch between q and the cache")
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    _check(q, "q", BF16)
    _check(k_cache, "k_cache", BF16, device=q.device)
    _check(v_cache, "v_cache", BF16, device=q.device)
    _check(block_table, "block_table", torch.int32, device=q.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == num_seqs, "block_table must be [seqs, max_blocks]")
    _check(seq_lens, "seq_lens", torch.int32, num_seqs, q.device)
    _check(partial_o, "partial_o", torch.float32, num_seqs * num_splits * n_q * hd, q.device)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, q.device)
    if out is None:
        out = torch.empty((num_seqs, n_q, hd), dtype=BF16, device=q.device)
    _check(out, "out", BF16, num_seqs * n_q * hd, q.device)
    call("smx_splitkv_decode_merged", _stream(q), q.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), partial_o.data_ptr(),
         partial_lse.data_ptr(), out.data_ptr(), num_seqs, num_splits,
         block_table.shape[1], num_blocks, bs, n_q, n_kv, hd, float(scale))
    return out


def lse_merge(partial_o: torch.Tensor, partial_lse: torch.Tensor,
              out: torch.Tensor | None = None) -> torch.Tensor:
    _need(partial_o.dim() == 4, "partial_o must be [seqs, splits, n_q, hd]")
    num_seqs, num_splits, n_q, hd = partial_o.shape
    _check(partial_o, "partial_o", torch.float32)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, partial_o.device)
    if out is None:
        out = torch.empty((num_seqs, n_q, hd), dtype=BF16, device=partial_o.device)
    _check(out, "out", BF16, num_seqs * n_q * hd, partial_o.device)
    call("smx_lse_merge", _stream(partial_o), partial_o.data_ptr(), partial_lse.data_ptr(),
         out.data_ptr(), num_seqs, num_splits, n_q, hd)
    return out


PLAN_WORDS = 64  # uint32 words per split-plan record (SMX_SPLITKV_PLAN_WORDS)


def splitkv_plan(seq_lens: torch.Tensor, block_table: torch.Tensor, block_size: int,
                 num_items: int, partial_o: torch.Tensor, partial_lse: torch.Tensor,
                 positions: torch.Tensor | None = None, slot_mapping: torch.Tensor | None = None,
                 plan: torch.Tensor | None = None) -> torch.Tensor:
    """Per-sequence split plan from the live lengths (device-side; one call
    per decode step serves every layer).  partial_o [seqs, num_splits, n_q,
    hd] / partial_lse fix num_splits and must be the buffers the planned
    attention calls use: slots no split writes are cleared here.  Returns
    the plan, int32 [num_items + seqs, PLAN_WORDS] (uint32 words)."""
    num_seqs = seq_lens.numel()
    _need(partial_o.dim() == 4 and partial_o.shape[0] == num_seqs,
          "partial_o must be [seqs, splits, n_q, hd]")
    _, num_splits, n_q, hd = partial_o.shape
    _check(seq_lens, "seq_lens", torch.int32, num_seqs)
    _check(block_table, "block_table", torch.int32, device=seq_lens.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == num_seqs, "block_table must be [seqs, max_blocks]")
    _check(partial_o, "partial_o", torch.float32, device=seq_lens.device)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, seq_lens.device)
    for t, name in ((positions, "positions"), (slot_mapping, "slot_mapping")):
        if t is not None:
            _check(t, name, torch.int64, num_seqs, seq_lens.device)
    nrec = num_items + num_seqs
    if plan is None:
        plan = torch.empty((nrec, PLAN_WORDS), dtype=torch.int32, device=seq_lens.device)
    _check(plan, "plan", torch.int32, nrec * PLAN_WORDS, seq_lens.device)
    call("smx_splitkv_plan", _stream(seq_lens), seq_lens.data_ptr(), _ptr(positions),
         _ptr(slot_mapping), block_table.data_ptr(), plan.data_ptr(), partial_o.data_ptr(),
         partial_lse.data_ptr(), num_seqs, num_items, num_splits, block_table.shape[1],
         block_size, n_q, hd)
    return plan


def splitkv_decode_planned_merged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                  block_table: torch.Tensor, plan: torch.Tensor, num_items: int,
                                  scale: float, partial_o: torch.Tensor, partial_lse: torch.Tensor,
                                  out: torch.Tensor | None = None) -> torch.Tensor:
    """splitkv_decode_merged over the splits of a plan (splitkv_plan with the
    same block table, num_items and partial buffers)."""
    _need(q.dim() == 3 and k_cache.dim() == 4, "q must be [seqs, n_q, hd], caches 4-D")
    num_seqs, n_q, hd = q.shape
    num_blocks, bs, n_kv, hd2 = k_cache.shape
    _need(hd == hd2, "head_dim mismatch between q and the cache")
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    _check(q, "q", BF16)
    _check(k_cache, "k_cache", BF16, device=q.device)
    _check(v_cache, "v_cache", BF16, device=q.device)
    _check(block_table, "block_table", torch.int32, device=q.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == num_seqs, "block_table must be [seqs, max_blocks]")
    _check(plan, "plan", torch.int32, (num_items + num_seqs) * PLAN_WORDS, q.device)
    _need(partial_o.dim() == 4 and partial_o.shape[0] == num_seqs, "partial_o must be [seqs, splits, n_q, hd]")
    num_splits = partial_o.shape[1]
    _check(partial_o, "partial_o", torch.float32, num_seqs * num_splits * n_q * hd, q.device)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, q.device)
    if out is None:
        out = torch.empty((num_seqs, n_q, hd), dtype=BF16, device=q.device)
    _check(out, "out", BF16, num_seqs * n_q * hd, q.device)
    call("smx_splitkv_decode_planned_merged", _stream(q), q.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), block_table.data_ptr(), plan.data_ptr(), partial_o.data_ptr(),
         partial_lse.data_ptr(), out.data_ptr(), num_seqs, num_items, num_splits,
         block_table.shape[1], num_blocks, bs, n_q, n_kv, hd, float(scale))
    return out


def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor | None, gamma: torch.Tensor, eps: float,
                out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None):
    """Returns (y, residual_out).  With residual=None: y = RMSNorm(x), residual_out = x."""
    _need(x.dim() >= 1, "x must have a hidden dimension")
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    _check(x, "x", BF16)
    _check(gamma, "gamma", BF16, hidden, x.device)
    if residual is not None:
        _check(residual, "residual", BF16, x.numel(), x.device)
    if out is None:
        out = torch.empty_like(x)
    _check(out, "out", BF16, x.numel(), x.device)
    if residual is not None and residual_out is None:
        residual_out = torch.empty_like(x)
    if residual_out is not None:
        _check(residual_out, "residual_out", BF16, x.numel(), x.device)
    call("smx_add_rmsnorm", _stream(x), x.data_ptr(),
         residual.data_ptr() if residual is not None else None, gamma.data_ptr(), out.data_ptr(),
         residual_out.data_ptr() if residual_out is not None else None, rows, hidden, float(eps))
    return out, (residual_out if residual is not None else x)


def qknorm_rope_kv_write(qkv: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor,
                         cos_sin: torch.Tensor, positions: torch.Tensor, slot_mapping: torch.Tensor,
                         k_cache: torch.Tensor, v_cache: torch.Tensor, n_q: int, n_kv: int,
                         eps: float, q_out: torch.Tensor | None = None) -> torch.Tensor:
    num_blocks, bs, n_kv2, hd = k_cache.shape
    _need(n_kv2 == n_kv, "cache kv-head count mismatch")
    num_tokens = positions.numel()
    _check(qkv, "qkv", BF16, num_tokens * (n_q + 2 * n_kv) * hd)
    _check(q_gamma, "q_gamma", BF16, hd, qkv.device)
    _check(k_gamma, "k_gamma", BF16, hd, qkv.device)
    _check(cos_sin, "cos_sin", BF16, device=qkv.device)
    _need(cos_sin.dim() == 2 and cos_sin.shape[1] == hd, "cos_sin must be [max_position, head_dim]")
    _check(positions, "positions", torch.int64, num_tokens, qkv.device)
    _check(slot_mapping, "slot_mapping", torch.int64, num_tokens, qkv.device)
    _check(k_cache, "k_cache", BF16, device=qkv.device)
    _check(v_cache, "v_cache", BF16, device=qkv.device)
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    if q_out is None:
        q_out = torch.empty((num_tokens, n_q, hd), dtype=BF16, device=qkv.device)
    _check(q_out, "q_out", BF16, num_tokens * n_q * hd, qkv.device)
    call("smx_qknorm_rope_kv_write", _stream(qkv), qkv.data_ptr(), q_gamma.data_ptr(),
         k_gamma.data_ptr(), cos_sin.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
         q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), num_tokens, n_q, n_kv, hd,
         num_blocks, bs, cos_sin.shape[0], float(eps))
    return q_out


def _gated_mul(gate_up, out, lut):
    _check(gate_up, "gate_up", BF16)
    d2 = gate_up.shape[-1]
    _need(d2 % 2 == 0, "last dimension must be even")
    rows = gate_up.numel() // d2
    if out is None:
        out = torch.empty((*gate_up.shape[:-1], d2 // 2), dtype=BF16, device=gate_up.device)
    _check(out, "out", BF16, rows * d2 // 2, gate_up.device)
    if lut is None:
        call("smx_silu_mul", _stream(gate_up), gate_up.data_ptr(), out.data_ptr(), rows, d2 // 2)
    else:
        call("smx_gelu_mul", _stream(gate_up), gate_up.data_ptr(),
             _lut_checked(lut, gate_up.device), out.data_ptr(), rows, d2 // 2)
    return out


def silu_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    return _gated_mul(gate_up, out, None)


def gelu_mul(gate_up: torch.Tensor, lut: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """The table GELU (gelu_table) of a [..., 2d] gate|up tensor times up."""
    return _gated_mul(gate_up, out, lut)


def embedding(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _check(table, "table", BF16)
    _need(table.dim() == 2, "table must be [vocab, hidden]")
    _check(ids, "ids", torch.int64, device=table.device)
    vocab, hidden = table.shape
    if out is None:
        out = torch.empty((ids.numel(), hidden), dtype=BF16, device=table.device)
    _check(out, "out", BF16, ids.numel() * hidden, table.device)
    call("smx_embedding", _stream(table), table.data_ptr(), ids.data_ptr(), out.data_ptr(),
         ids.numel(), vocab, hidden)
    return out


#: rows up to which the two-launch argmax is the faster one: more rows fill the
#: chip with one workgroup each (vocab 65536 / 151936 in a graph, two launches
#: against one: 32 rows 8.1 / 9.2 us, 8.4 / 11.9; 64 rows 10.7 / 12.6, 8.5 / 12.3;
#: 256 rows 26.9 / 31.9, 9.5 / 19.5)
ARGMAX_PARTS_ROWS = 32
#: vocab above which it is also for a call that allocates the keys, about 2.5 us of
#: the host's time (eager, one row, allocating against one launch: 65536 8.4 us, 7.3;
#: 98304 8.5, 7.6; 110000 8.6, 9.2; 151936 8.3, 8.8)
ARGMAX_ALLOC_VOCAB = 98304


def argmax_num_keys(rows: int, vocab: int) -> int:
    """Elements of the `keys` workspace argmax() takes; 0 where it uses none."""
    return rows * load().smx_argmax_parts(vocab) if 1 <= rows <= ARGMAX_PARTS_ROWS else 0


def argmax(logits: torch.Tensor, out: torch.Tensor | None = None,
           keys: torch.Tensor | None = None) -> torch.Tensor:
    """Greedy token of each row.  A few long rows take two launches with a
    workspace between them: `keys` (int64, argmax_num_keys elements), or above
    ARGMAX_ALLOC_VOCAB one allocated here.  With `out` and no `keys` the call allocates nothing, as a recorded
    step must not, and the row takes one launch."""
    _check(logits, "logits", BF16)
    vocab = logits.shape[-1]
    rows = logits.numel() // vocab
    num_keys = argmax_num_keys(rows, vocab)
    if keys is not None:
        _check(keys, "keys", torch.int64, num_keys, logits.device)
    elif num_keys and out is None and vocab > ARGMAX_ALLOC_VOCAB:
        keys = torch.empty((num_keys,), dtype=torch.int64, device=logits.device)
    if out is None:
        out = torch.empty((rows,), dtype=torch.int64, device=logits.device)
    _check(out, "out", torch.int64, rows, logits.device)
    if num_keys and keys is not None:
        call("smx_argmax_bf16_parts", _stream(logits), logits.data_ptr(), rows, vocab,
             keys.data_ptr(), num_keys, out.data_ptr())
        return out
    call("smx_argmax_bf16", _stream(logits), logits.data_ptr(), rows, vocab, out.data_ptr())
    return out


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """key, value: [num_tokens, n_kv, head_dim]; caches [blocks, bs, n_kv, head_dim]."""
    num_blocks, bs, n_kv, hd = k_cache.shape
    num_tokens = slot_mapping.numel()
    _check(key, "key", BF16, num_tokens * n_kv * hd)
    _check(value, "value", BF16, num_tokens * n_kv * hd, key.device)
    _check(k_cache, "k_cache", BF16, device=key.device)
    _check(v_cache, "v_cache", BF16, device=key.device)
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    _check(slot_mapping, "slot_mapping", torch.int64, num_tokens, key.device)
    call("smx_reshape_and_cache", _stream(key), key.data_ptr(), value.data_ptr(),
         k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), num_tokens, n_kv, hd,
         num_blocks, bs)


def decode_advance(next_ids: torch.Tensor, ids: torch.Tensor, positions: torch.Tensor,
                   seq_lens: torch.Tensor, slot_mapping: torch.Tensor, block_table: torch.Tensor,
                   block_size: int, tokens_out: torch.Tensor | None = None,
                   forced_ids: torch.Tensor | None = None,
                   forced_len: torch.Tensor | None = None,
                   argmax_keys: torch.Tensor | None = None,
                   embed_table: torch.Tensor | None = None,
                   embed_out: torch.Tensor | None = None) -> None:
    """forced_ids [rows, max_len] int64 with forced_len [rows] int32 on the
    device; tokens_out [rows, max_len] int64 (same max_len); argmax_keys
    [rows, num_keys] int64 from add_rmsnorm_gemv_argmax (next_ids is then
    written with the argmax); embed_table [vocab, hidden] bf16 with embed_out
    [rows, hidden]: the embedding rows of the new ids for the next step."""
    rows = ids.numel()
    _check(next_ids, "next_ids", torch.int64, rows)
    _check(ids, "ids", torch.int64, rows, next_ids.device)
    _check(positions, "positions", torch.int64, rows, next_ids.device)
    _check(seq_lens, "seq_lens", torch.int32, rows, next_ids.device)
    _check(slot_mapping, "slot_mapping", torch.int64, rows, next_ids.device)
    _check(block_table, "block_table", torch.int32, device=next_ids.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == rows, "block_table must be [rows, max_blocks]")
    _need((forced_ids is None) == (forced_len is None), "forced_ids and forced_len go together")
    max_len = 0
    for name, t in (("tokens_out", tokens_out), ("forced_ids", forced_ids)):
        if t is not None:
            _check(t, name, torch.int64, device=next_ids.device)
            _need(t.dim() == 2 and t.shape[0] == rows, f"{name} must be [rows, max_len]")
            _need(max_len in (0, t.shape[1]), "tokens_out and forced_ids need the same max_len")
            max_len = t.shape[1]
    if forced_len is not None:
        _check(forced_len, "forced_len", torch.int32, rows, next_ids.device)
    num_keys = 0
    if argmax_keys is not None:
        _check(argmax_keys, "argmax_keys", torch.int64, device=next_ids.device)
        _need(argmax_keys.dim() == 2 and argmax_keys.shape[0] == rows, "argmax_keys must be [rows, n]")
        num_keys = argmax_keys.shape[1]
    _need((embed_table is None) == (embed_out is None), "embed_table and embed_out go together")
    vocab = hidden = 0
    if embed_table is not None:
        _check(embed_table, "embed_table", BF16, device=next_ids.device)
        _need(embed_table.dim() == 2, "embed_table must be [vocab, hidden]")
        vocab, hidden = embed_table.shape
        _check(embed_out, "embed_out", BF16, rows * hidden, next_ids.device)
    call("smx_decode_advance", _stream(ids), next_ids.data_ptr(),
         argmax_keys.data_ptr() if argmax_keys is not None else None, num_keys,
         forced_ids.data_ptr() if forced_ids is not None else None,
         forced_len.data_ptr() if forced_len is not None else None, ids.data_ptr(),
         positions.data_ptr(), seq_lens.data_ptr(), slot_mapping.data_ptr(), block_table.data_ptr(),
         tokens_out.data_ptr() if tokens_out is not None else None, rows, block_table.shape[1],
         block_size, max_len, _ptr(embed_table), _ptr(embed_out), vocab, hidden)


def _norm_gemv_checks(x, residual, gamma, residual_out, k):
    _check(x, "x", BF16, k)
    _check(gamma, "gamma", BF16, k, x.device)
    if residual is not None:
        _check(residual, "residual", BF16, k, x.device)
    if residual_out is not None:
        _check(residual_out, "residual_out", BF16, k, x.device)
        _need(residual_out.data_ptr() not in (x.data_ptr(),
                                               residual.data_ptr() if residual is not None else -1),
              "residual_out must not alias x or residual")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def add_rmsnorm_gemv(x: torch.Tensor, residual: torch.Tensor | None, gamma: torch.Tensor,
                     w: torch.Tensor, n: int, k: int, eps: float,
                     residual_out: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """y = W . (RMSNorm(x + residual) * gamma); residual_out = bf16(x + residual)."""
    _norm_gemv_checks(x, residual, gamma, residual_out, k)
    _check(w, "w", torch.uint8, n * q4_0_row_bytes(k), x.device)
    if out is None:
        out = torch.empty((1, n), dtype=BF16, device=x.device)
    _check(out, "out", BF16, n, x.device)
    call("smx_q4_0_add_rmsnorm_gemv", _stream(x), x.data_ptr(), _ptr(residual), gamma.data_ptr(),
         _ptr(residual_out), w.data_ptr(), out.data_ptr(), n, k, float(eps))
    return out


def add_rmsnorm_gemv_swiglu(x: torch.Tensor, residual: torch.Tensor | None, gamma: torch.Tensor,
                            w: torch.Tensor, d: int, k: int, eps: float,
                            residual_out: torch.Tensor | None = None,
                            out: torch.Tensor | None = None,
                            lut: torch.Tensor | None = None) -> torch.Tensor:
    """add+RMSNorm, gate/up GEMV and SwiGLU -- or, given the GELU table
    (gelu_table) as lut, the reference's table GELU in place of SiLU."""
    _norm_gemv_checks(x, residual, gamma, residual_out, k)
    _check(w, "w", torch.uint8, 2 * d * q4_0_row_bytes(k), x.device)
    if out is None:
        out = torch.empty((1, d), dtype=BF16, device=x.device)
    _check(out, "out", BF16, d, x.device)
    if lut is None:
        call("smx_q4_0_add_rmsnorm_gemv_swiglu", _stream(x), x.data_ptr(), _ptr(residual),
             gamma.data_ptr(), _ptr(residual_out), w.data_ptr(), out.data_ptr(), d, k, float(eps))
    else:
        call("smx_q4_0_add_rmsnorm_gemv_gelu", _stream(x), x.data_ptr(), _ptr(residual),
             gamma.data_ptr(), _ptr(residual_out), w.data_ptr(), _lut_checked(lut, x.device),
             out.data_ptr(), d, k, float(eps))
    return out


def add_rmsnorm_gemv_gelu(x: torch.Tensor, residual: torch.Tensor | None, gamma: torch.Tensor,
                          w: torch.Tensor, lut: torch.Tensor, d: int, k: int, eps: float,
                          residual_out: torch.Tensor | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """NativeUp.execute as one launch: add+RMSNorm, gate/up GEMV, table GELU."""
    return add_rmsnorm_gemv_swiglu(x, residual, gamma, w, d, k, eps, residual_out, out, lut)


def argmax_keys_size(n: int, k: int) -> int:
    return int(load().smx_q4_0_argmax_keys_size(n, k))


def add_rmsnorm_gemv_argmax(x: torch.Tensor, residual: torch.Tensor | None, gamma: torch.Tensor,
                            w: torch.Tensor, n: int, k: int, eps: float, keys: torch.Tensor,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits = W . RMSNorm(x + residual) * gamma, plus per-workgroup argmax
    keys [argmax_keys_size(n, k)] int64 for decode_advance."""
    _norm_gemv_checks(x, residual, gamma, None, k)
    _check(w, "w", torch.uint8, n * q4_0_row_bytes(k), x.device)
    _check(keys, "keys", torch.int64, device=x.device)
    if out is None:
        out = torch.empty((1, n), dtype=BF16, device=x.device)
    _check(out, "out", BF16, n, x.device)
    call("smx_q4_0_add_rmsnorm_gemv_argmax", _stream(x), x.data_ptr(), _ptr(residual),
         gamma.data_ptr(), w.data_ptr(), out.data_ptr(), keys.data_ptr(), keys.numel(), n, k,
         float(eps))
    return out


def qknorm_rope_splitkv_decode_merged(qkv: torch.Tensor, q_gamma: torch.Tensor,
                                      k_gamma: torch.Tensor, cos_sin: torch.Tensor,
                                      positions: torch.Tensor, slot_mapping: torch.Tensor,
                                      k_cache: torch.Tensor, v_cache: torch.Tensor,
                                      block_table: torch.Tensor, seq_lens: torch.Tensor,
                                      num_splits: int, scale: float, eps: float, n_q: int,
                                      partial_o: torch.Tensor, partial_lse: torch.Tensor,
                                      out: torch.Tensor | None = None) -> torch.Tensor:
    """q/k RMSNorm + RoPE + KV write + split-KV decode + merge for one decode
    token per sequence (qkv: raw QKV projection [num_seqs, (n_q+2n_kv)*hd])."""
    num_blocks, bs, n_kv, hd = k_cache.shape
    num_seqs = seq_lens.numel()
    _check(qkv, "qkv", BF16, num_seqs * (n_q + 2 * n_kv) * hd)
    _check(q_gamma, "q_gamma", BF16, hd, qkv.device)
    _check(k_gamma, "k_gamma", BF16, hd, qkv.device)
    _check(cos_sin, "cos_sin", BF16, device=qkv.device)
    _need(cos_sin.dim() == 2 and cos_sin.shape[1] == hd, "cos_sin must be [max_position, head_dim]")
    _check(positions, "positions", torch.int64, num_seqs, qkv.device)
    _check(slot_mapping, "slot_mapping", torch.int64, num_seqs, qkv.device)
    _check(k_cache, "k_cache", BF16, device=qkv.device)
    _check(v_cache, "v_cache", BF16, device=qkv.device)
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    _check(block_table, "block_table", torch.int32, device=qkv.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == num_seqs, "block_table must be [seqs, max_blocks]")
    _check(seq_lens, "seq_lens", torch.int32, num_seqs, qkv.device)
    _check(partial_o, "partial_o", torch.float32, num_seqs * num_splits * n_q * hd, qkv.device)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, qkv.device)
    if out is None:
        out = torch.empty((num_seqs, n_q, hd), dtype=BF16, device=qkv.device)
    _check(out, "out", BF16, num_seqs * n_q * hd, qkv.device)
    call("smx_qknorm_rope_splitkv_decode_merged", _stream(qkv), qkv.data_ptr(), q_gamma.data_ptr(),
         k_gamma.data_ptr(), cos_sin.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
         k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
         partial_o.data_ptr(), partial_lse.data_ptr(), out.data_ptr(), num_seqs, num_splits,
         block_table.shape[1], num_blocks, bs, n_q, n_kv, hd, cos_sin.shape[0], float(eps),
         float(scale))
    return out


def qknorm_rope_splitkv_decode_planned_merged(qkv: torch.Tensor, q_gamma: torch.Tensor,
                                              k_gamma: torch.Tensor, cos_sin: torch.Tensor,
                                              k_cache: torch.Tensor, v_cache: torch.Tensor,
                                              block_table: torch.Tensor, plan: torch.Tensor,
                                              num_items: int, scale: float, eps: float, n_q: int,
                                              partial_o: torch.Tensor, partial_lse: torch.Tensor,
                                              out: torch.Tensor | None = None) -> torch.Tensor:
    """qknorm_rope_splitkv_decode_merged over the splits of a plan; the
    positions and slots come from the plan (splitkv_plan given them)."""
    num_blocks, bs, n_kv, hd = k_cache.shape
    num_seqs = block_table.shape[0]
    _check(qkv, "qkv", BF16, num_seqs * (n_q + 2 * n_kv) * hd)
    _check(q_gamma, "q_gamma", BF16, hd, qkv.device)
    _check(k_gamma, "k_gamma", BF16, hd, qkv.device)
    _check(cos_sin, "cos_sin", BF16, device=qkv.device)
    _need(cos_sin.dim() == 2 and cos_sin.shape[1] == hd, "cos_sin must be [max_position, head_dim]")
    _check(k_cache, "k_cache", BF16, device=qkv.device)
    _check(v_cache, "v_cache", BF16, device=qkv.device)
    _need(v_cache.shape == k_cache.shape, "k_cache and v_cache shapes differ")
    _check(block_table, "block_table", torch.int32, device=qkv.device)
    _need(block_table.dim() == 2, "block_table must be [seqs, max_blocks]")
    _check(plan, "plan", torch.int32, (num_items + num_seqs) * PLAN_WORDS, qkv.device)
    _need(partial_o.dim() == 4 and partial_o.shape[0] == num_seqs, "partial_o must be [seqs, splits, n_q, hd]")
    num_splits = partial_o.shape[1]
    _check(partial_o, "partial_o", torch.float32, num_seqs * num_splits * n_q * hd, qkv.device)
    _check(partial_lse, "partial_lse", torch.float32, num_seqs * num_splits * n_q, qkv.device)
    if out is None:
        out = torch.empty((num_seqs, n_q, hd), dtype=BF16, device=qkv.device)
    _check(out, "out", BF16, num_seqs * n_q * hd, qkv.device)
    call("smx_qknorm_rope_splitkv_decode_planned_merged", _stream(qkv), qkv.data_ptr(),
         q_gamma.data_ptr(), k_gamma.data_ptr(), cos_sin.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), block_table.data_ptr(), plan.data_ptr(), partial_o.data_ptr(),
         partial_lse.data_ptr(), out.data_ptr(), num_seqs, num_items, num_splits,
         block_table.shape[1], num_blocks, bs, n_q, n_kv, hd, cos_sin.shape[0], float(eps),
         float(scale))
    return out


def compute_slot_mapping(query_start_loc: torch.Tensor, positions: torch.Tensor,
                         block_table: torch.Tensor, block_size: int, max_tokens: int | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """int64 slots [max_tokens] of a ragged batch (-1 for padding and for
    positions past the block table)."""
    num_reqs = query_start_loc.numel() - 1
    _need(num_reqs >= 1, "query_start_loc needs num_reqs + 1 entries")
    _check(query_start_loc, "query_start_loc", torch.int32)
    _need(positions.dtype == torch.int64 and positions.device == query_start_loc.device
          and positions.is_contiguous(), "positions must be contiguous int64 on the same device")
    _check(block_table, "block_table", torch.int32, device=query_start_loc.device)
    _need(block_table.dim() == 2 and block_table.shape[0] >= num_reqs, "block_table must be [reqs, max_blocks]")
    num_tokens = positions.numel()
    max_tokens = num_tokens if max_tokens is None else max_tokens
    if out is None:
        out = torch.empty(max(max_tokens, 1), dtype=torch.int64, device=positions.device)
    _check(out, "out", torch.int64, device=positions.device)
    _need(out.numel() >= max_tokens, "out must hold max_tokens entries")
    pos_ptr = positions.data_ptr() if num_tokens else out.data_ptr()  # never read when empty
    call("smx_compute_slot_mapping", _stream(out), query_start_loc.data_ptr(), num_reqs,
         pos_ptr, block_table.data_ptr(), out.data_ptr(), num_tokens,
         max(max_tokens, 1), block_table.shape[1], block_size)
    return out


def _plain(t: torch.Tensor, dtype: torch.dtype, index: int) -> bool:
    """Whether t is a contiguous `dtype` tensor on GPU `index` (get_device() is -1 on
    the CPU): half of _check's time for the calls that a step makes of small work,
    with _check only to say what is wrong."""
    return t.dtype is dtype and t.get_device() == index and t.is_contiguous()


def _all_plain(index: int, dtype: torch.dtype, **tensors: torch.Tensor) -> None:
    """Refuses the first of `tensors` that is not _plain."""
    for name, t in tensors.items():
        _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
        if index < 0 or not _plain(t, dtype, index):
            _check(t, name, dtype, device=torch.device("cuda", max(index, 0)))
            raise ValueError(f"{name} is not a valid argument")


def _rows_checks(q, k_cache, v_cache, block_table, seq_lens, workspace, out):
    """The checks the row attentions share -> (out, allocated if None; sizes).  (Written
    out: a dozen calls of _need are 0.4 us of these calls' seven.)"""
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dtype is BF16 and q.dim() == 3):
        raise ValueError("q must be a bf16 GPU tensor [tokens, n_q, hd]")
    tokens, n_q, hd = q.shape
    step, head_step, unit = q.stride()
    if tokens < 1 or n_q < 1:
        raise ValueError("q must hold a token and a head")
    if tokens == 1:
        step = n_q * hd
    if not (unit == 1 and (n_q == 1 or head_step == hd) and step >= n_q * hd):
        raise ValueError("a token's heads must be contiguous in q and its tokens apart")
    if not (q.data_ptr() % 16 == 0 and step % 8 == 0):
        raise ValueError("q's tokens must be 16-byte aligned")
    i = q.get_device()
    if not (_plain(k_cache, BF16, i) and _plain(v_cache, BF16, i)
            and _plain(block_table, torch.int32, i) and _plain(seq_lens, torch.int32, i)):
        _all_plain(i, BF16, k_cache=k_cache, v_cache=v_cache)
        _all_plain(i, torch.int32, block_table=block_table, seq_lens=seq_lens)
    shape = k_cache.shape
    if not (len(shape) == 4 and v_cache.shape == shape):
        raise ValueError("the caches must be [blocks, block_size, n_kv, hd], both alike")
    num_blocks, bs, n_kv, cache_hd = shape
    if hd != cache_hd:
        raise ValueError("head_dim mismatch between q and the cache")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [seqs, max_blocks]")
    num_seqs, max_blocks = block_table.shape
    if seq_lens.numel() != num_seqs:
        raise ValueError("seq_lens must have an entry for each row of block_table")
    if workspace is not None and not _plain(workspace, torch.uint8, i):
        _all_plain(i, torch.uint8, workspace=workspace)
    if out is None:
        # (empty_like: 0.9 us, an empty of the sizes 1.5)
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(
            (tokens, n_q, hd), dtype=BF16, device=q.device)
    elif not _plain(out, BF16, i):
        _all_plain(i, BF16, out=out)
    if out.numel() != tokens * n_q * hd:
        raise ValueError("out must have q's elements")
    return out, step, (num_seqs, max_blocks, num_blocks, bs, n_q, n_kv, hd)


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def prompt_attention_workspace(q: torch.Tensor, k_cache: torch.Tensor,
                               block_table: torch.Tensor) -> torch.Tensor | None:
    """The workspace prompt_attention uses for these sizes (uint8; None where it
    uses none).  Calls that can overlap need one each."""
    _, bs, n_kv, hd = k_cache.shape
    return _workspace(load().smx_prompt_attention_workspace(
        q.shape[0], block_table.shape[0], block_table.shape[1], bs, q.shape[1], n_kv, hd),
        q.device)


def prompt_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     block_table: torch.Tensor, query_start_loc: torch.Tensor,
                     seq_lens: torch.Tensor, scale: float,
                     workspace: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed query rows over the paged cache.  q [tokens, n_q,
    hd] (tokens may be strided, a slice of the QKV rows); sequence r's queries
    are the rows query_start_loc[r]..query_start_loc[r + 1] and the last of its
    seq_lens[r] tokens, whose K and V the cache holds.  Rows of no sequence are
    left as they are in `out`.  Without `workspace` (prompt_attention_workspace)
    one is allocated where the call needs it."""
    out, step, sizes = _rows_checks(q, k_cache, v_cache, block_table, seq_lens, workspace, out)
    if not _plain(query_start_loc, torch.int32, q.get_device()):
        _all_plain(q.get_device(), torch.int32, query_start_loc=query_start_loc)
    if query_start_loc.numel() != sizes[0] + 1:
        raise ValueError("query_start_loc must have num_seqs + 1 entries")
    args = (_stream(q), q.data_ptr(), step, k_cache.data_ptr(), v_cache.data_ptr(),
            block_table.data_ptr(), query_start_loc.data_ptr(), seq_lens.data_ptr())
    rest = (out.data_ptr(), q.shape[0], *sizes, float(scale))
    if workspace is None:
        # most prompts need none: the call that refuses is cheaper than asking each time
        try:
            call("smx_prompt_attention", *args, None, 0, *rest)
            return out
        except SmxError as e:
            workspace = prompt_attention_workspace(q, k_cache, block_table)
            if e.code != SMX_EINVAL or workspace is None:
                raise
    call("smx_prompt_attention", *args, workspace.data_ptr(), workspace.numel(), *rest)
    return out


def shared_prefix_attention_workspace(q: torch.Tensor, k_cache: torch.Tensor,
                                      prefix_table: torch.Tensor,
                                      block_table: torch.Tensor) -> torch.Tensor | None:
    """The workspace shared_prefix_attention uses for these sizes (uint8)."""
    _, bs, n_kv, hd = k_cache.shape
    return _workspace(load().smx_shared_prefix_attention_workspace(
        q.shape[0], prefix_table.numel(), block_table.shape[1], bs, q.shape[1], n_kv, hd),
        q.device)


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_len: torch.Tensor,
                            block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                            workspace: torch.Tensor | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of sequences that share their first prefix_len[0] tokens
    (pages prefix_table, int32 [blocks]), read once for all.  q [seqs, n_q, hd];
    block_table [seqs, max_blocks] by absolute position (its entries below the
    prefix are not used); seq_lens the whole lengths, prefix included."""
    out, step, sizes = _rows_checks(q, k_cache, v_cache, block_table, seq_lens, workspace, out)
    if q.shape[0] != sizes[0]:
        raise ValueError("q must have a row for each sequence of block_table")
    i = q.get_device()
    if not (_plain(prefix_table, torch.int32, i) and _plain(prefix_len, torch.int32, i)):
        _all_plain(i, torch.int32, prefix_table=prefix_table, prefix_len=prefix_len)
    if not (prefix_table.dim() == 1 and prefix_table.numel() >= 1):
        raise ValueError("prefix_table must be [prefix_blocks]")
    if prefix_len.numel() != 1:
        raise ValueError("prefix_len must have 1 element")
    if workspace is None:
        workspace = shared_prefix_attention_workspace(q, k_cache, prefix_table, block_table)
    call("smx_shared_prefix_attention", _stream(q), q.data_ptr(), step, k_cache.data_ptr(),
         v_cache.data_ptr(), prefix_table.data_ptr(), prefix_len.data_ptr(),
         block_table.data_ptr(), seq_lens.data_ptr(), _ptr(workspace),
         workspace.numel() if workspace is not None else 0, out.data_ptr(), sizes[0],
         prefix_table.numel(), *sizes[1:], float(scale))
    return out


class RequestTables:
    """What request_tables() writes besides the block table; the buffers are checked
    once, here.
      num_pages        int32 [reqs]: pages each request now has
      free_count       int32 [1]: pages left in the free list
      query_start_loc  int32 [reqs + 1]
      seq_lens         int32 [reqs]
      positions        int64 [max_tokens], 0 past the last token
      slot_mapping     int64 [max_tokens], -1 past the last token"""

    __slots__ = ("num_pages", "free_count", "query_start_loc", "seq_lens", "positions",
                 "slot_mapping", "reqs", "max_tokens", "index")

    def __init__(self, num_pages, free_count, query_start_loc, seq_lens, positions,
                 slot_mapping):
        _check(num_pages, "num_pages", torch.int32)
        reqs, dev = num_pages.numel(), num_pages.device
        _check(free_count, "free_count", torch.int32, 1, dev)
        _check(query_start_loc, "query_start_loc", torch.int32, reqs + 1, dev)
        _check(seq_lens, "seq_lens", torch.int32, reqs, dev)
        _check(positions, "positions", torch.int64, device=dev)
        _check(slot_mapping, "slot_mapping", torch.int64, positions.numel(), dev)
        _need(reqs >= 1 and positions.numel() >= 1, "there must be a request and a token")
        self.num_pages, self.free_count = num_pages, free_count
        self.query_start_loc, self.seq_lens = query_start_loc, seq_lens
        self.positions, self.slot_mapping = positions, slot_mapping
        self.reqs, self.max_tokens, self.index = reqs, positions.numel(), num_pages.get_device()

    def replace(self, **buffers) -> "RequestTables":
        """The same with some buffers others."""
        return RequestTables(**{**{n: getattr(self, n) for n in self.__slots__[:6]}, **buffers})


def request_tables_out(num_pages: torch.Tensor, max_tokens: int) -> RequestTables:
    """Buffers for request_tables(out=...).  A program that keeps its pages in
    place takes .replace(num_pages=num_pages, free_count=free_count) of it."""
    _need(max_tokens >= 1, "max_tokens must be >= 1")
    reqs, dev = num_pages.numel(), num_pages.device
    i32 = dict(dtype=torch.int32, device=dev)
    i64 = dict(dtype=torch.int64, device=dev)
    return RequestTables(torch.empty(reqs, **i32), torch.empty(1, **i32),
                         torch.empty(reqs + 1, **i32), torch.empty(reqs, **i32),
                         torch.empty(max_tokens, **i64), torch.empty(max_tokens, **i64))


def _pages_checks(num_pages, free_pages, free_count, block_table, lens, lens_name):
    if not isinstance(num_pages, torch.Tensor):
        raise ValueError("num_pages must be a tensor")
    i = num_pages.get_device()
    if i < 0 or not (_plain(num_pages, torch.int32, i) and _plain(free_pages, torch.int32, i)
                     and _plain(free_count, torch.int32, i)
                     and _plain(block_table, torch.int32, i) and _plain(lens, torch.int32, i)):
        _all_plain(i, torch.int32, num_pages=num_pages, free_pages=free_pages,
                   free_count=free_count, block_table=block_table, **{lens_name: lens})
    reqs = num_pages.numel()
    if not (reqs >= 1 and lens.numel() == reqs):
        raise ValueError(f"{lens_name} must have an entry for each request")
    if free_pages.numel() < 1:
        raise ValueError("free_pages must have room for a page")
    if free_count.numel() != 1:
        raise ValueError("free_count must have 1 element")
    shape = block_table.shape
    if not (len(shape) == 2 and shape[0] == reqs and shape[1] >= 1):
        raise ValueError("block_table must be [reqs, max_blocks]")
    return reqs, shape[1], i


def request_tables(query_lens: torch.Tensor, context_lens: torch.Tensor,
                   num_pages: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                   block_table: torch.Tensor, block_size: int, max_tokens: int | None = None,
                   out: RequestTables | None = None) -> RequestTables:
    """A step's block tables, offsets, lengths, positions and slots from the
    requests' new and cached token counts, on the device.  Pages that block_table's
    rows lack are taken from the end of the free list and written into the table;
    num_pages and free_count are updated out of place, or in place where `out`
    holds them.  max_tokens (without `out`): the size of positions and slots."""
    reqs, max_blocks, i = _pages_checks(num_pages, free_pages, free_count, block_table,
                                        query_lens, "query_lens")
    if not (isinstance(context_lens, torch.Tensor) and _plain(context_lens, torch.int32, i)
            and context_lens.numel() == reqs):
        _check(context_lens, "context_lens", torch.int32, reqs, num_pages.device)
    if out is None:
        if max_tokens is None:
            raise ValueError("max_tokens or out is needed")
        out = request_tables_out(num_pages, max_tokens)
    if not (isinstance(out, RequestTables) and out.reqs == reqs and out.index == i
            and max_tokens in (None, out.max_tokens)):
        raise ValueError("out must be RequestTables of these requests and max_tokens")
    call("smx_request_tables", _stream(num_pages), query_lens.data_ptr(),
         context_lens.data_ptr(), num_pages.data_ptr(), free_pages.data_ptr(),
         free_count.data_ptr(), block_table.data_ptr(), out.num_pages.data_ptr(),
         out.free_count.data_ptr(), out.query_start_loc.data_ptr(), out.seq_lens.data_ptr(),
         out.positions.data_ptr(), out.slot_mapping.data_ptr(), reqs, out.max_tokens, max_blocks,
         free_pages.numel(), block_size)
    return out


def release_pages(keep_lens: torch.Tensor, num_pages: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, block_table: torch.Tensor, block_size: int) -> None:
    """Give the pages beyond the first keep_lens[r] tokens of every request back to
    the free list (0: all of a finished request's; fewer than its length: those
    of rejected tokens).  Everything is updated in place.  A page belongs to one
    request: one that several rows list would be in the free list several times."""
    reqs, max_blocks, _ = _pages_checks(num_pages, free_pages, free_count, block_table, keep_lens,
                                        "keep_lens")
    call("smx_release_pages", _stream(num_pages), keep_lens.data_ptr(), num_pages.data_ptr(),
         free_pages.data_ptr(), free_count.data_ptr(), block_table.data_ptr(), reqs, max_blocks,
         free_pages.numel(), block_size)


class Q4KVCache:
    """A paged KV cache held in 4 bits (smx_q4_reshape_and_cache): blocks of 32 channels of
    a token's head share an fp16 scale d and hold codes of 0..15 for d * (code - 8).
      codes   uint8 [2, num_blocks, n_kv, block_size, head_dim / 2], K first
      scales  fp16 [2, num_blocks, n_kv, block_size, head_dim / 32]
    4.5 bits a value.  The order of a row's codes is the kernels' own: q4_kv_read gives
    the values."""

    __slots__ = ("codes", "scales", "num_blocks", "n_kv", "block_size", "head_dim", "index")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        _check(codes, "codes", torch.uint8)
        _need(codes.dim() == 5 and codes.shape[0] == 2,
              "codes must be [2, num_blocks, n_kv, block_size, head_dim / 2]")
        _, self.num_blocks, self.n_kv, self.block_size, half = codes.shape
        self.head_dim = 2 * half
        _need(self.head_dim in (64, 128), "head_dim must be 64 or 128")
        _check(scales, "scales", torch.float16, device=codes.device)
        _need(scales.shape == (*codes.shape[:4], half // 16),
              "scales must be [2, num_blocks, n_kv, block_size, head_dim / 32]")
        self.codes, self.scales, self.index = codes, scales, codes.get_device()

    def planes(self) -> list[torch.Tensor]:
        """The tensors of a PageSet(page_dim=1)."""
        return [self.codes, self.scales]


def q4_kv_cache(num_blocks: int, block_size: int, n_kv: int, head_dim: int,
                device) -> Q4KVCache:
    """An empty cache in 4 bits."""
    _need(min(num_blocks, n_kv) >= 1, "num_blocks and n_kv must be >= 1")
    _need(32 <= block_size <= 4096 and block_size & (block_size - 1) == 0,
          "block_size must be a power of two in [32, 4096]")
    _need(head_dim in (64, 128), "head_dim must be 64 or 128")
    shape = (2, num_blocks, n_kv, block_size)
    return Q4KVCache(torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device),
                     torch.zeros((*shape, head_dim // 32), dtype=torch.float16, device=device))


def _q4_cache(cache, index: int) -> Q4KVCache:
    if not isinstance(cache, Q4KVCache):
        raise ValueError("cache must be a Q4KVCache")
    if cache.index != index:
        raise ValueError("the cache must be on the other tensors' device")
    return cache


def reshape_and_cache_q4(key: torch.Tensor, value: torch.Tensor, cache: Q4KVCache,
                         slot_mapping: torch.Tensor) -> None:
    """reshape_and_cache into a cache in 4 bits.  key, value [tokens, n_kv, hd]: a token's
    heads are contiguous, tokens may be strided (a slice of the QKV rows).  A slot is given
    once in a call."""
    _need(isinstance(slot_mapping, torch.Tensor), "slot_mapping must be a tensor")
    i = slot_mapping.get_device()
    c = _q4_cache(cache, i)
    _check(slot_mapping, "slot_mapping", torch.int64)
    tokens = slot_mapping.numel()
    steps = []
    for t, name in ((key, "key"), (value, "value")):
        if not (isinstance(t, torch.Tensor) and t.dtype is BF16 and t.get_device() == i):
            raise ValueError(f"{name} must be a bf16 tensor on slot_mapping's device")
        if tuple(t.shape) != (tokens, c.n_kv, c.head_dim):
            raise ValueError(f"{name} must be [tokens, n_kv, head_dim]")
        step, head_step, unit = t.stride()
        if not (unit == 1 and (c.n_kv == 1 or head_step == c.head_dim)):
            raise ValueError(f"a token's heads must be contiguous in {name}")
        if tokens <= 1:
            step = c.n_kv * c.head_dim
        if step < c.n_kv * c.head_dim or step % 8 or t.data_ptr() % 16:
            raise ValueError(f"{name}'s tokens must be apart and 16-byte aligned")
        steps.append(step)
    if tokens == 0:
        return
    call("smx_q4_reshape_and_cache", _stream(slot_mapping), key.data_ptr(), steps[0],
         value.data_ptr(), steps[1], c.codes.data_ptr(), c.scales.data_ptr(),
         slot_mapping.data_ptr(), tokens, c.n_kv, c.head_dim, c.num_blocks, c.block_size)


def q4_kv_read(cache: Q4KVCache, slot_mapping: torch.Tensor,
               out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """The (key, value) that a cache in 4 bits holds for the tokens at slot_mapping, exactly:
    fp32 [tokens, n_kv, hd]; 0 for slots outside it."""
    _check(slot_mapping, "slot_mapping", torch.int64)
    c = _q4_cache(cache, slot_mapping.get_device())
    shape = (slot_mapping.numel(), c.n_kv, c.head_dim)
    n = shape[0] * shape[1] * shape[2]
    if out is None:
        first = torch.empty(shape, dtype=torch.float32, device=slot_mapping.device)
        out = first, first.new_empty(shape)
    else:
        for t, name in zip(out, ("out[0]", "out[1]")):
            _check(t, name, torch.float32, n, slot_mapping.device)
    if n:
        call("smx_q4_kv_read", _stream(slot_mapping), c.codes.data_ptr(), c.scales.data_ptr(),
             slot_mapping.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), *shape, c.num_blocks,
             c.block_size)
    return out


def qknorm_rope_kv_write_q4(qkv: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor,
                            cos_sin: torch.Tensor, positions: torch.Tensor,
                            slot_mapping: torch.Tensor, cache: Q4KVCache, n_q: int, n_kv: int,
                            eps: float, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """qknorm_rope_kv_write into a cache in 4 bits."""
    _check(positions, "positions", torch.int64)
    dev = positions.device
    c = _q4_cache(cache, positions.get_device())
    _need(c.n_kv == n_kv, "cache kv-head count mismatch")
    hd, num_tokens = c.head_dim, positions.numel()
    _check(qkv, "qkv", BF16, num_tokens * (n_q + 2 * n_kv) * hd, dev)
    _check(q_gamma, "q_gamma", BF16, hd, dev)
    _check(k_gamma, "k_gamma", BF16, hd, dev)
    _check(cos_sin, "cos_sin", BF16, device=dev)
    _need(cos_sin.dim() == 2 and cos_sin.shape[1] == hd, "cos_sin must be [max_position, head_dim]")
    _check(slot_mapping, "slot_mapping", torch.int64, num_tokens, dev)
    if q_out is None:
        q_out = torch.empty((num_tokens, n_q, hd), dtype=BF16, device=dev)
    _check(q_out, "q_out", BF16, num_tokens * n_q * hd, dev)
    call("smx_q4_qknorm_rope_kv_write", _stream(positions), qkv.data_ptr(), q_gamma.data_ptr(),
         k_gamma.data_ptr(), cos_sin.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
         q_out.data_ptr(), c.codes.data_ptr(), c.scales.data_ptr(), num_tokens, n_q, n_kv, hd,
         c.num_blocks, c.block_size, cos_sin.shape[0], float(eps))
    return q_out


def q4_attention_workspace(q: torch.Tensor, cache: Q4KVCache, block_table: torch.Tensor,
                           query_start_loc: torch.Tensor | None = None) -> torch.Tensor | None:
    """The workspace q4_attention uses for these sizes (uint8; None where it uses none),
    with or without offsets.  Calls that can overlap need one each."""
    return _workspace(load().smx_q4_attention_workspace(
        q.shape[0], block_table.shape[0], block_table.shape[1], cache.block_size, q.shape[1],
        cache.n_kv, cache.head_dim), q.device)


def q4_attention(q: torch.Tensor, cache: Q4KVCache, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, scale: float,
                 query_start_loc: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """prompt_attention over a cache in 4 bits: sequence r's queries are the rows
    query_start_loc[r]..query_start_loc[r + 1] of q [tokens, n_q, hd] (tokens may be
    strided), the last of its seq_lens[r] tokens.  Without query_start_loc row r is
    sequence r's newest token: a decode step.  Weights are rounded to fp16, and of
    prompts the cache's values.  Rows of no sequence are left as they are in
    `out`.  Without `workspace` (q4_attention_workspace) one is allocated where the call
    needs it."""
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dtype is BF16 and q.dim() == 3):
        raise ValueError("q must be a bf16 GPU tensor [tokens, n_q, hd]")
    tokens, n_q, hd = q.shape
    step, head_step, unit = q.stride()
    if tokens < 1 or n_q < 1:
        raise ValueError("q must hold a token and a head")
    if tokens == 1:
        step = n_q * hd
    if not (unit == 1 and (n_q == 1 or head_step == hd) and step >= n_q * hd):
        raise ValueError("a token's heads must be contiguous in q and its tokens apart")
    if q.data_ptr() % 16 or step % 8:
        raise ValueError("q's tokens must be 16-byte aligned")
    i = q.get_device()
    c = _q4_cache(cache, i)
    if hd != c.head_dim:
        raise ValueError("head_dim mismatch between q and the cache")
    _all_plain(i, torch.int32, block_table=block_table, seq_lens=seq_lens)
    if block_table.dim() != 2:
        raise ValueError("block_table must be [seqs, max_blocks]")
    num_seqs, max_blocks = block_table.shape
    if seq_lens.numel() != num_seqs:
        raise ValueError("seq_lens must have an entry for each row of block_table")
    if query_start_loc is None:
        if tokens != num_seqs:
            raise ValueError("without query_start_loc q must have a row for each sequence")
    else:
        _all_plain(i, torch.int32, query_start_loc=query_start_loc)
        if query_start_loc.numel() != num_seqs + 1:
            raise ValueError("query_start_loc must have num_seqs + 1 entries")
    if out is None:
        out = torch.empty((tokens, n_q, hd), dtype=BF16, device=q.device)
    else:
        _all_plain(i, BF16, out=out)
        if out.numel() != tokens * n_q * hd:
            raise ValueError("out must have q's elements")
    if workspace is None:
        workspace = q4_attention_workspace(q, c, block_table, query_start_loc)
    else:
        _all_plain(i, torch.uint8, workspace=workspace)
    call("smx_q4_attention", _stream(q), q.data_ptr(), step, c.codes.data_ptr(),
         c.scales.data_ptr(), block_table.data_ptr(), _ptr(query_start_loc), seq_lens.data_ptr(),
         _ptr(workspace), workspace.numel() if workspace is not None else 0, out.data_ptr(),
         tokens, num_seqs, max_blocks, c.num_blocks, c.block_size, n_q, c.n_kv, hd, float(scale))
    return out


def _made(cls, *tensors):
    """A `cls` of tensors that this module has allocated, without the checks of its
    constructor (a microsecond or two of calls of four)."""
    x = object.__new__(cls)
    for name, t in zip(cls.__slots__, tensors):
        setattr(x, name, t)
    return x


class BeamSelection:
    """What beam_select() writes, [seqs, width], the best first:
      parents  int32: the row of logits it continues, -1 where there is none
      tokens   int64, -1 where there is none
      scores   fp32, -inf where there is none"""

    __slots__ = ("parents", "tokens", "scores")

    def __init__(self, parents, tokens, scores):
        _check(parents, "parents", torch.int32)
        _need(parents.dim() == 2, "parents must be [seqs, width]")
        _check(tokens, "tokens", torch.int64, parents.numel(), parents.device)
        _check(scores, "scores", torch.float32, parents.numel(), parents.device)
        _need(tokens.shape == parents.shape and scores.shape == parents.shape,
              "parents, tokens and scores must be [seqs, width]")
        self.parents, self.tokens, self.scores = parents, tokens, scores


def beam_select_out(seqs: int, width: int, device) -> BeamSelection:
    """Buffers for beam_select(out=...)."""
    return _made(BeamSelection, torch.empty((seqs, width), dtype=torch.int32, device=device),
                 torch.empty((seqs, width), dtype=torch.int64, device=device),
                 torch.empty((seqs, width), dtype=torch.float32, device=device))


def beam_select_workspace(logits: torch.Tensor, beams: int, width: int) -> torch.Tensor | None:
    """The workspace beam_select uses for these sizes (uint8).  Calls that can overlap need
    one each."""
    return _workspace(load().smx_beam_select_workspace(
        logits.shape[0] // max(beams, 1), beams, width, logits.shape[1], logits.element_size()),
        logits.device)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, beams: int, width: int,
                done: torch.Tensor | None = None, pad_id: int = 0,
                workspace: torch.Tensor | None = None,
                out: BeamSelection | None = None) -> BeamSelection:
    """The `width` best continuations of each sequence's `beams` rows of logits [seqs *
    beams, vocab] (bf16 or fp32; rows may be strided) by scores[row] + log softmax(logits
    [row]), scores fp32 [rows]: in order, ties to the lowest beam and token.  Logits of
    -inf and NaN are never chosen, rows whose score is -inf offer nothing.  A row that is
    done (bool [rows]) offers pad_id at its own score.  Without `workspace`
    (beam_select_workspace) one is allocated."""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() == 2
            and logits.dtype in (BF16, torch.float32)):
        raise ValueError("logits must be a bf16 or fp32 GPU tensor [rows, vocab]")
    rows, vocab = logits.shape
    step, unit = logits.stride()
    if not (1 <= beams <= 64 and 1 <= width <= 64):
        raise ValueError("beams and width must be in [1, 64]")
    if rows < 1 or rows % beams or vocab < 1:
        raise ValueError("logits must have `beams` rows for each sequence")
    if rows == 1:
        step = vocab
    if not ((unit == 1 or vocab == 1) and step >= vocab):
        raise ValueError("a row's logits must be contiguous and rows apart")
    i = logits.get_device()
    _all_plain(i, torch.float32, scores=scores)
    if scores.numel() != rows:
        raise ValueError("scores must have an entry for each row of logits")
    if done is not None:
        _all_plain(i, torch.bool, done=done)
        if done.numel() != rows:
            raise ValueError("done must have an entry for each row of logits")
    if not 0 <= pad_id < vocab:
        raise ValueError("pad_id must be a token")
    if out is None:
        out = beam_select_out(rows // beams, width, logits.device)
    elif not (isinstance(out, BeamSelection) and out.parents.shape == (rows // beams, width)
              and out.parents.get_device() == i):
        raise ValueError("out must be a BeamSelection of these sequences and width")
    if workspace is None:
        workspace = beam_select_workspace(logits, beams, width)
    else:
        _all_plain(i, torch.uint8, workspace=workspace)
    call("smx_beam_select", _stream(logits), logits.data_ptr(), step, logits.element_size(),
         scores.data_ptr(), _ptr(done), workspace.data_ptr(), workspace.numel(),
         out.parents.data_ptr(), out.tokens.data_ptr(), out.scores.data_ptr(), rows // beams,
         beams, width, vocab, pad_id)
    return out


class ForkedPages:
    """What fork_pages() writes:
      block_table  int32 [rows, max_blocks], -1 past a row's pages
      num_pages    int32 [rows]
      lens         int32 [rows]
      free_pages   int32 [any]: the free list, -1 past its end
      free_count   int32 [1]
      copies       int32 [rows, 2]: (page, its copy) for copy_pages, else -1"""

    __slots__ = ("block_table", "num_pages", "lens", "free_pages", "free_count", "copies")

    def __init__(self, block_table, num_pages, lens, free_pages, free_count, copies):
        _check(block_table, "block_table", torch.int32)
        _need(block_table.dim() == 2, "block_table must be [rows, max_blocks]")
        rows, dev = block_table.shape[0], block_table.device
        _check(num_pages, "num_pages", torch.int32, rows, dev)
        _check(lens, "lens", torch.int32, rows, dev)
        _check(free_pages, "free_pages", torch.int32, device=dev)
        _check(free_count, "free_count", torch.int32, 1, dev)
        _check(copies, "copies", torch.int32, 2 * rows, dev)
        self.block_table, self.num_pages, self.lens = block_table, num_pages, lens
        self.free_pages, self.free_count, self.copies = free_pages, free_count, copies


def fork_pages_out(block_table: torch.Tensor, free_pages: torch.Tensor) -> ForkedPages:
    """Buffers for fork_pages(out=...) of a table and free list of these sizes."""
    _check(block_table, "block_table", torch.int32)
    _check(free_pages, "free_pages", torch.int32, device=block_table.device)
    _need(block_table.dim() == 2, "block_table must be [rows, max_blocks]")
    return _forked_pages(block_table, free_pages)


def _forked_pages(block_table, free_pages):
    new, rows = block_table.new_empty, block_table.shape[0]
    return _made(ForkedPages, new(block_table.shape), new(rows), new(rows),
                 new(free_pages.shape), new(1), new((rows, 2)))


def fork_pages(parents: torch.Tensor, lens: torch.Tensor, num_pages: torch.Tensor,
               free_pages: torch.Tensor, free_count: torch.Tensor, block_table: torch.Tensor,
               num_blocks: int, block_size: int, out: ForkedPages | None = None) -> ForkedPages:
    """Block tables of the rows that a step goes on with: new row j continues the first
    lens[parents[j]] tokens of old row parents[j] (outside the rows: it is empty).  Rows of
    one parent share its pages, but for a last page that is not full: the first child keeps
    it, the others get pages from the end of the free list, into which copy_pages(...,
    copies) copies it before they are written.  Pages that no new row lists are free again.
    A row whose copy finds no page is cut to its whole pages (see lens).  int32 throughout;
    `out` may hold free_pages and free_count themselves, the rest is apart from the inputs."""
    reqs, max_blocks, i = _pages_checks(num_pages, free_pages, free_count, block_table, lens,
                                        "lens")
    _all_plain(i, torch.int32, parents=parents)
    if parents.numel() != reqs:
        raise ValueError("parents must have an entry for each row of block_table")
    if out is None:
        out = _forked_pages(block_table, free_pages)
    elif not (isinstance(out, ForkedPages) and out.block_table.shape == block_table.shape
              and out.free_pages.numel() == free_pages.numel()
              and out.block_table.get_device() == i):
        raise ValueError("out must be ForkedPages of this table and free list")
    call("smx_fork_pages", _stream(num_pages), parents.data_ptr(), lens.data_ptr(),
         num_pages.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
         block_table.data_ptr(), out.block_table.data_ptr(), out.num_pages.data_ptr(),
         out.lens.data_ptr(), out.free_pages.data_ptr(), out.free_count.data_ptr(),
         out.copies.data_ptr(), reqs, max_blocks, num_blocks, free_pages.numel(), block_size)
    return out


class CompactedPages:
    """What compact_pages() writes:
      block_table  int32 [rows, max_blocks], -1 past a row's pages
      free_pages   int32 [num_blocks]: the free list, -1 past its end
      free_count   int32 [1]
      moves        int32 [num_blocks // 2, 2]: (from, to) for copy_pages, then -1"""

    __slots__ = ("block_table", "free_pages", "free_count", "moves")

    def __init__(self, block_table, free_pages, free_count, moves):
        _check(block_table, "block_table", torch.int32)
        _need(block_table.dim() == 2, "block_table must be [rows, max_blocks]")
        dev = block_table.device
        _check(free_pages, "free_pages", torch.int32, device=dev)
        _check(free_count, "free_count", torch.int32, 1, dev)
        _check(moves, "moves", torch.int32, free_pages.numel() // 2 * 2, dev)
        self.block_table, self.free_pages = block_table, free_pages
        self.free_count, self.moves = free_count, moves


def compact_pages(num_pages: torch.Tensor, block_table: torch.Tensor, num_blocks: int,
                  out: CompactedPages | None = None) -> CompactedPages:
    """Moves the pages that block_table's rows list (each its num_pages first entries; rows
    may share pages) to the front of the pool: the table with the new places, the free
    list of all pages behind them, and the moves for copy_pages, which must be done before
    the table is used.  `out` may hold block_table itself."""
    _need(isinstance(num_pages, torch.Tensor), "num_pages must be a tensor")
    i = num_pages.get_device()
    _all_plain(i, torch.int32, num_pages=num_pages, block_table=block_table)
    rows = num_pages.numel()
    if not (block_table.dim() == 2 and block_table.shape[0] == rows >= 1
            and block_table.shape[1] >= 1):
        raise ValueError("block_table must be [rows, max_blocks]")
    _need(num_blocks >= 2, "num_blocks must be >= 2")
    if out is None:
        new = num_pages.new_empty
        out = _made(CompactedPages, new(block_table.shape), new(num_blocks), new(1),
                    new((num_blocks // 2, 2)))
    elif not (isinstance(out, CompactedPages) and out.block_table.shape == block_table.shape
              and out.free_pages.numel() == num_blocks and out.block_table.get_device() == i):
        raise ValueError("out must be CompactedPages of this table and num_blocks")
    call("smx_compact_pages", _stream(num_pages), num_pages.data_ptr(), block_table.data_ptr(),
         out.block_table.data_ptr(), out.free_pages.data_ptr(), out.free_count.data_ptr(),
         out.moves.data_ptr(), rows, block_table.shape[1], num_blocks)
    return out


class PageSet:
    """The caches whose pages copy_pages copies together: tensors on one GPU whose
    dimension page_dim counts the pages ([2, num_blocks, ...] caches: 1), as many in each.
    Built once; it keeps the tensors."""

    __slots__ = ("tensors", "planes", "num_planes", "page_bytes", "num_blocks", "index")

    def __init__(self, tensors: list[torch.Tensor], page_dim: int = 1):
        _need(len(tensors) >= 1, "there must be a tensor")
        planes, self.num_blocks = [], None
        for n, t in enumerate(tensors):
            _need(isinstance(t, torch.Tensor), f"tensors[{n}] must be a tensor")
            _check(t, f"tensors[{n}]", t.dtype, device=tensors[0].device)
            _need(0 <= page_dim < t.dim() and t.numel() > 0,
                  f"tensors[{n}] must have pages in dimension {page_dim}")
            pages = t.shape[page_dim]
            self.num_blocks = pages if self.num_blocks is None else self.num_blocks
            _need(pages == self.num_blocks, "the tensors must have as many pages each")
            size = t.element_size() * t.stride(page_dim)
            _need(size % 16 == 0 and t.data_ptr() % 16 == 0,
                  f"tensors[{n}]'s pages must be whole and aligned 16 bytes")
            count = t.numel() * t.element_size() // (size * pages)
            planes += [[t.data_ptr() + k * size * pages, size] for k in range(count)]
        self.tensors = list(tensors)
        self.planes = torch.tensor(planes, dtype=torch.int64).to(tensors[0].device)
        self.num_planes, self.page_bytes = len(planes), max(b for _, b in planes)
        self.index = tensors[0].get_device()


def copy_pages(pages: PageSet, pairs: torch.Tensor) -> None:
    """Copies page src to page dst of every cache of `pages` for each row (src, dst) of
    pairs (int32 [n, 2]); rows with an entry outside the pool are skipped.  No page may be
    the dst of two rows, or the dst of one and the src of another."""
    if not isinstance(pages, PageSet):
        raise ValueError("pages must be a PageSet")
    _all_plain(pages.index, torch.int32, pairs=pairs)
    if not (pairs.dim() == 2 and pairs.shape[1] == 2):
        raise ValueError("pairs must be [n, 2]")
    if pairs.shape[0]:
        call("smx_copy_pages", _stream(pairs), pages.planes.data_ptr(), pages.num_planes,
             pages.page_bytes, pairs.data_ptr(), pairs.shape[0], pages.num_blocks)


class PackedQ4_0:
    """A Q4_0 matrix in the packed layout of the MFMA GEMMs (smx_q4_0_repack):
    ``data`` uint8 [packed_bytes], the [n, k] matrix it holds (gated: the
    [2n, k] gate|up matrix, n = d).  q4_0_gemm, q4_0_gemm_swiglu and
    q4_0_gemm_argmax take one in place of the GGUF tensor."""

    __slots__ = ("data", "n", "k", "gated")

    def __init__(self, data: torch.Tensor, n: int, k: int, gated: bool):
        self.data, self.n, self.k, self.gated = data, int(n), int(k), bool(gated)


def q4_0_packed_bytes(n: int, k: int, gated: bool = False) -> int:
    """Bytes of the packed form of an [n, k] Q4_0 matrix (gated: [2n, k]);
    -1 when unsupported (k not a positive multiple of 256)."""
    return int(load().smx_q4_0_packed_bytes(n, k, 1 if gated else 0))


def q4_0_repack(w: torch.Tensor, n: int, k: int, gated: bool = False,
                out: torch.Tensor | None = None) -> PackedQ4_0:
    """Repack GGUF Q4_0 weights (n rows; gated: the 2n gate|up rows) into the
    packed layout; lossless (the same codes and fp16 scales, moved)."""
    nbytes = q4_0_packed_bytes(n, k, gated)
    _need(nbytes > 0, "the packed layout needs k a positive multiple of 256")
    _check(w, "w", torch.uint8, (2 * n if gated else n) * q4_0_row_bytes(k))
    if out is None:
        out = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
    _check(out, "out", torch.uint8, nbytes, w.device)
    _need(out.data_ptr() % 16 == 0, "out must be 16-byte aligned")
    call("smx_q4_0_repack", _stream(w), w.data_ptr(), out.data_ptr(), n, k, 1 if gated else 0)
    return PackedQ4_0(out, n, k, gated)


def _gemm_x(x: torch.Tensor, k: int, align: int) -> None:
    _need(x.dim() == 2 and x.shape[1] == k and 1 <= x.shape[0] <= 16, "x must be [m <= 16, k]")
    _check(x, "x", BF16)
    if x.data_ptr() % align:
        raise ValueError(f"x must be {align}-byte aligned")


def _packed_checked(w: PackedQ4_0, n: int, k: int, gated: bool, device) -> int:
    if not (w.n == n and w.k == k and w.gated == gated):
        raise ValueError(f"packed weights hold [{w.n}, {w.k}] (gated={w.gated}), the call wants "
                         f"[{n}, {k}] (gated={gated})")
    _check(w.data, "w.data", torch.uint8, q4_0_packed_bytes(n, k, gated), device)
    return w.data.data_ptr()


def q4_0_gemm(x: torch.Tensor, w: torch.Tensor | PackedQ4_0, n: int, k: int,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """y [m, n] = x [m, k] . W^T for m <= 16 rows (MFMA kernel); W GGUF Q4_0
    or packed (q4_0_repack)."""
    packed = isinstance(w, PackedQ4_0)
    _gemm_x(x, k, 16 if packed else 8)
    if out is None:
        out = torch.empty((x.shape[0], n), dtype=BF16, device=x.device)
    _check(out, "out", BF16, x.shape[0] * n, x.device)
    if packed:
        call("smx_q4_0_gemm_packed", _stream(x), x.data_ptr(),
             _packed_checked(w, n, k, False, x.device), out.data_ptr(), x.shape[0], n, k)
    else:
        _check(w, "w", torch.uint8, n * q4_0_row_bytes(k), x.device)
        call("smx_q4_0_gemm", _stream(x), x.data_ptr(), w.data_ptr(), out.data_ptr(),
             x.shape[0], n, k)
    return out


def q4_0_gemm_rows(x: torch.Tensor, w: torch.Tensor, n: int, k: int,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """y [m, n] = x [m, k] . W^T for any m >= 1 and any k % 32 == 0, W GGUF Q4_0
    (m <= 16: the exact weights; more rows: their bf16 roundings)."""
    _need(k % 32 == 0 and k > 0 and n > 0, "need n > 0 and k a positive multiple of 32")
    _need(x.dim() == 2 and x.shape[0] >= 1 and x.shape[1] == k, "x must be [m, k]")
    _check(x, "x", BF16)
    _need(x.data_ptr() % 16 == 0, "x must be 16-byte aligned")
    _check(w, "w", torch.uint8, n * q4_0_row_bytes(k), x.device)
    if out is None:
        out = torch.empty((x.shape[0], n), dtype=BF16, device=x.device)
    _check(out, "out", BF16, x.shape[0] * n, x.device)
    call("smx_q4_0_gemm_rows", _stream(x), x.data_ptr(), w.data_ptr(), out.data_ptr(),
         x.shape[0], n, k)
    return out


def gemm_rows_preferred(m: int, n: int, k: int) -> bool:
    """Whether q4_0_gemm_rows beats dequantisation + a library GEMM (m > 16)."""
    return bool(load().smx_q4_0_gemm_rows_preferred(m, n, k))


def q4_0_gemm_swiglu(x: torch.Tensor, w: torch.Tensor | PackedQ4_0, d: int, k: int,
                     out: torch.Tensor | None = None,
                     lut: torch.Tensor | None = None) -> torch.Tensor:
    """out [m, d] = silu(x W_gate^T) * (x W_up^T), W = [gate; up] [2d, k] (GGUF
    Q4_0, or packed gated by q4_0_repack); given the GELU table (gelu_table)
    as lut, the table GELU in place of SiLU."""
    packed = isinstance(w, PackedQ4_0)
    _gemm_x(x, k, 16 if packed else 8)
    if out is None:
        out = torch.empty((x.shape[0], d), dtype=BF16, device=x.device)
    _check(out, "out", BF16, x.shape[0] * d, x.device)
    if packed:
        wp = _packed_checked(w, d, k, True, x.device)
        if lut is None:
            call("smx_q4_0_gemm_packed_swiglu", _stream(x), x.data_ptr(), wp, out.data_ptr(),
                 x.shape[0], d, k)
        else:
            call("smx_q4_0_gemm_packed_gelu", _stream(x), x.data_ptr(), wp,
                 _lut_checked(lut, x.device), out.data_ptr(), x.shape[0], d, k)
        return out
    _check(w, "w", torch.uint8, 2 * d * q4_0_row_bytes(k), x.device)
    if lut is None:
        call("smx_q4_0_gemm_swiglu", _stream(x), x.data_ptr(), w.data_ptr(), out.data_ptr(),
             x.shape[0], d, k)
    else:
        call("smx_q4_0_gemm_gelu", _stream(x), x.data_ptr(), w.data_ptr(),
             _lut_checked(lut, x.device), out.data_ptr(), x.shape[0], d, k)
    return out


def q4_0_gemm_gelu(x: torch.Tensor, w: torch.Tensor | PackedQ4_0, lut: torch.Tensor, d: int, k: int,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    return q4_0_gemm_swiglu(x, w, d, k, out, lut)


def gemm_keys_per_row(n: int) -> int:
    """Greedy-argmax keys q4_0_gemm_argmax writes per row (one per 16 outputs)."""
    return int(load().smx_q4_0_gemm_keys_per_row(n))


def q4_0_gemm_argmax(x: torch.Tensor, w: torch.Tensor | PackedQ4_0, n: int, k: int,
                     keys: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x W^T (m <= 16 rows; W GGUF Q4_0 or packed) plus keys [m, ceil(n / 16)]
    int64 (uint64 bits), the greedy-argmax keys decode_advance(argmax_keys=keys)
    reduces."""
    _gemm_x(x, k, 16)
    m = x.shape[0]
    _check(keys, "keys", torch.int64, m * gemm_keys_per_row(n), x.device)
    if out is None:
        out = torch.empty((m, n), dtype=BF16, device=x.device)
    _check(out, "out", BF16, m * n, x.device)
    if isinstance(w, PackedQ4_0):
        call("smx_q4_0_gemm_packed_argmax", _stream(x), x.data_ptr(),
             _packed_checked(w, n, k, False, x.device), out.data_ptr(), keys.data_ptr(), m, n, k)
    else:
        _check(w, "w", torch.uint8, n * q4_0_row_bytes(k), x.device)
        call("smx_q4_0_gemm_argmax", _stream(x), x.data_ptr(), w.data_ptr(), out.data_ptr(),
             keys.data_ptr(), m, n, k)
    return out
