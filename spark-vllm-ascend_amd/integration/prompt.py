"""One decoder layer over packed prompt rows: whole prompts, chunks behind what
the cache holds, or a few drafted tokens a sequence.

The reference hands such calls to vLLM's stock layer (attention,
post-attention norm, MLP and next norm for ``x.shape[0] != 1``,
src/spark_vllm_ascend/integration/model.py:50-61).  Here the layer is

  QKV linear -> q/k RMSNorm + RoPE + KV write -> causal attention of the packed
  rows over the paged cache (torch_ops.prompt_attention) -> o_proj linear ->
  add + RMSNorm(post norm) -> gate|up linear -> SwiGLU or table GELU -> down
  linear

with the linears' products by their quant method (any number of rows).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ..native import torch_ops


@dataclass
class PromptRows:
    """Where the rows of a pass stand: row t of sequence r (query_start_loc[r] <= t <
    query_start_loc[r + 1]) is one of the last tokens of its seq_lens[r]."""
    block_table: torch.Tensor       # int32 [seqs, max_blocks]
    query_start_loc: torch.Tensor   # int32 [seqs + 1]
    seq_lens: torch.Tensor          # int32 [seqs], these rows included
    positions: torch.Tensor         # int64 [rows]
    slot_mapping: torch.Tensor      # int64 [rows], -1: K and V are not kept
    workspace: torch.Tensor | None = None  # prompt_attention's, for all layers


def prompt_layer(cfg, layer, cos_sin: torch.Tensor, scale: float,
                 act_lut: torch.Tensor | None, x: torch.Tensor, residual: torch.Tensor,
                 rows: PromptRows) -> tuple[torch.Tensor, torch.Tensor]:
    """(down projection's output, residual after the attention add) of the rows x
    bf16 [T, hidden], normalised by the layer's input norm; the rows' K and V are
    written to the layer's cache."""
    c, L, ops = cfg, layer, torch_ops
    kc, vc = L.kv_cache[0], L.kv_cache[1]
    qkv = L.qkv.quant_method.apply(L.qkv, x)
    q = ops.qknorm_rope_kv_write(qkv, L.q_norm, L.k_norm, cos_sin, rows.positions,
                                 rows.slot_mapping, kc, vc, c.n_q, c.n_kv, c.eps)
    # rows of no sequence (padding) are left as they are: zeros here
    attn = ops.prompt_attention(q, kc, vc, rows.block_table, rows.query_start_loc, rows.seq_lens,
                                scale, workspace=rows.workspace, out=torch.zeros_like(q))
    o = L.o_proj.quant_method.apply(L.o_proj, attn.view(x.shape[0], -1))
    h, residual = ops.add_rmsnorm(o, residual, L.post_norm, c.eps)
    gate_up = L.gate_up.quant_method.apply(L.gate_up, h)
    act = ops.silu_mul(gate_up) if act_lut is None else ops.gelu_mul(gate_up, act_lut)
    return L.down.quant_method.apply(L.down, act), residual
