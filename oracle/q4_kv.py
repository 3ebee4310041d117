"""The KV cache held in 4 bits, for the oracle -- test infrastructure.

Restates the format of smx_q4_reshape_and_cache in numpy: blocks of 32 channels of one
head of a token with an fp16 scale d and codes of 0..15 for d * (code - 8), as the
reference's Q4_0 weights are stored (src/spark_vllm_ascend/integration/weights.py:34-40):
d = fp16(m / -8), m the first value of largest magnitude, code = floor(x / d + 8.5).
"""
from __future__ import annotations

import numpy as np

BLOCK = 32


def quantise(x: np.ndarray):
    """x [..., hd] -> (codes int64 [..., hd], d fp16 [..., hd / 32])."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, BLOCK)
    nan = np.isnan(b).any(-1)
    b = np.where(np.isnan(b), 0.0, b)
    at = np.abs(b).argmax(-1)[..., None]
    m = np.take_along_axis(b, at, -1)[..., 0]
    with np.errstate(all="ignore"):
        d = np.clip(m / -8, -65504.0, 65504.0).astype(np.float16)
        dd = d.astype(np.float64)[..., None]
        c = np.where(dd == 0, 8.0, np.floor(b / dd + 8.5))
    c = np.where(nan[..., None], 0, np.clip(c, 0, 15)).astype(np.int64)
    return c.reshape(x.shape), np.where(nan, np.float16(np.nan), d)


def values(codes: np.ndarray, d: np.ndarray) -> np.ndarray:
    """float64 values [..., hd]."""
    return (codes.astype(np.float64) - 8) * np.repeat(d.astype(np.float64), BLOCK, -1)


def key_order(hd: int) -> list[int]:
    """The channel of each half-byte of a K row (lowest first): dword g * (hd / 32) + b
    holds channels 32 b + 8 g + (0, 2, 4, 6, 1, 3, 5, 7).  V's are in channel order."""
    nb = hd // BLOCK
    return [BLOCK * (dw % nb) + 8 * (dw // nb) + i for dw in range(hd // 8)
            for i in (0, 2, 4, 6, 1, 3, 5, 7)]


def pack(codes: np.ndarray, is_key: bool) -> np.ndarray:
    """uint8 [..., hd / 2]"""
    c = codes[..., key_order(codes.shape[-1])] if is_key else codes
    return (c[..., 0::2] | c[..., 1::2] << 4).astype(np.uint8)


def unpack(rows: np.ndarray, is_key: bool) -> np.ndarray:
    """int64 codes [..., hd]"""
    c = np.stack((rows & 15, rows >> 4), -1).reshape(*rows.shape[:-1], -1).astype(np.int64)
    if is_key:
        out = np.empty_like(c)
        out[..., key_order(c.shape[-1])] = c
        return out
    return c


def plane_values(codes: np.ndarray, scales: np.ndarray, plane: int) -> np.ndarray:
    """A cache's K (0) or V (1) as float64 [blocks, block_size, n_kv, hd]."""
    v = values(unpack(codes[plane], plane == 0), scales[plane])
    return v.transpose(0, 2, 1, 3)
