"""The 4-bit paged KV cache: its format, in plain tensor operations (what the kernels are held to).

A pool is uint8 [blocks, kv heads, 2 (keys, values), 9 D] for a head dimension D of 64, 128 or 256; a block holds 16 tokens.  Every
64 channels of a row share a scale s and a low end lo (bf16) and have codes n of 4 bits:

    x  = the bf16 row, brought into +-32768
    lo = min x,   s = bf16((max x - lo) / 15),   n = clamp(rint((x - lo) / s), 0, 15)      (s = 0: n = 0)
    value = n s + lo

A group that holds a NaN has s = NaN.  4.5 bits a value: 9/16 of the fp8 cache's bytes.  Within a block the first 8 D bytes are code words
(32 bits, eight consecutive channels of a token, the first in the lowest bits) in the order of ``word_places``, the last D bytes the
pairs (s, lo) as [token][group].
"""
from __future__ import annotations

import torch

BLOCK = 16
GROUP = 64
LIMIT = 32768.0
HEAD_DIMS = (64, 128, 256)


def pool_shape(blocks: int, kv_heads: int, head_dim: int):
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"the 4-bit KV cache has head dimensions {HEAD_DIMS}, not {head_dim}")
    return (blocks, kv_heads, 2, 9 * head_dim)


def word_places(head_dim: int, values: bool, device="cpu") -> torch.Tensor:
    """[16, D / 8]: place of the word of channels 8 w .. 8 w + 7 of token t among a block's code words."""
    t = torch.arange(BLOCK, device=device)[:, None]
    w = torch.arange(head_dim // 8, device=device)[None, :]
    if values:
        g, j, p = w & 7, w >> 3, t >> 1
        if head_dim == 256:
            return t * 32 + (g ^ (t & 6)) * 4 + j
        if head_dim == 128:
            return p * 32 + (g ^ (t & 6)) * 4 + (t & 1) * 2 + j
        return p * 16 + (g ^ ((p & 2) << 1)) * 2 + (t & 1)
    c, j = w & 3, w >> 2
    if head_dim == 256:
        return t * 32 + ((j >> 2) ^ (t & 1)) * 16 + c * 4 + (j & 3)
    return t * (head_dim // 8) + c * (head_dim // 32) + j


def quantise(x: torch.Tensor):
    """bf16 rows [..., D] -> (codes int32 [..., D / 64, 64], s bf16, lo bf16 [..., D / 64])."""
    f = x.to(torch.bfloat16).float().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, GROUP))
    lo, hi = f.amin(-1), f.amax(-1)                       # (NaN where the group has one)
    s = ((hi - lo) / 15.0).to(torch.bfloat16)
    n = ((f - lo[..., None]) / s.float()[..., None]).round().clamp(0, 15)
    return torch.where(s.float()[..., None] > 0, n, 0.0).to(torch.int32), s, lo.to(torch.bfloat16)


def dequantise(n: torch.Tensor, s: torch.Tensor, lo: torch.Tensor) -> torch.Tensor:
    """fp32 values [..., D]."""
    return (n * s.float()[..., None] + lo.float()[..., None]).flatten(-2)


def round_trip(x: torch.Tensor) -> torch.Tensor:
    """What the cache makes of bf16 rows: fp32 values."""
    return dequantise(*quantise(x))


def write_rows(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor, tokens: torch.Tensor) -> None:
    """Rows [rows, kv heads, D] into (blocks[r], tokens[r]) of the pool, in place."""
    D = pool.shape[-1] // 9
    words = pool.view(torch.int32)
    head = torch.arange(pool.shape[1], device=pool.device)[None, :, None]
    at = blocks.long()[:, None, None]
    tok = tokens.long()
    for part, x in ((0, k), (1, v)):
        n, s, lo = quantise(x)
        bits = (n.flatten(-2).unflatten(-1, (-1, 8)).long() << (4 * torch.arange(8, device=n.device))).sum(-1)
        places = word_places(D, part == 1, pool.device)[tok]
        words[at, head, part, places[:, None, :]] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        pair = 2 * D + tok[:, None] * (D // GROUP) + torch.arange(D // GROUP, device=pool.device)
        words[at, head, part, pair[:, None, :]] = torch.stack([s, lo], -1).view(torch.int32)[..., 0]


def read_rows(pool: torch.Tensor, blocks: torch.Tensor, tokens: torch.Tensor):
    """(k, v) fp32 [rows, kv heads, D] at (blocks[r], tokens[r])."""
    D = pool.shape[-1] // 9
    words = pool.view(torch.int32)
    head = torch.arange(pool.shape[1], device=pool.device)[None, :, None]
    at = blocks.long()[:, None, None]
    tok = tokens.long()
    out = []
    for part in (0, 1):
        w = words[at, head, part, word_places(D, part == 1, pool.device)[tok][:, None, :]]
        n = (w[..., None] >> (4 * torch.arange(8, dtype=torch.int32, device=pool.device))) & 15
        pair = 2 * D + tok[:, None] * (D // GROUP) + torch.arange(D // GROUP, device=pool.device)
        p = words[at, head, part, pair[:, None, :]].contiguous().view(torch.bfloat16).unflatten(-1, (D // GROUP, 2))
        out.append(dequantise(n.flatten(-2).unflatten(-1, (-1, GROUP)), p[..., 0], p[..., 1]))
    return out[0], out[1]
