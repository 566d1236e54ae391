"""Attention over the visible keys of each query (sliding window, first tokens), in 64 bits, query row by query row.

Key t is visible to the query at position p iff t <= p and (window == 0 or t > p - window or t < sinks).  Keys that a
query does not see are left out of its sums altogether, so what they hold cannot matter; a row that sees nothing is
zero.  Block-scaled caches: element = e4m3 code * 2^(byte - 127), bytes per (block, 16 slots, kv head, K or V).
"""
from __future__ import annotations

import torch

from .attention import _as_u8, _E4M3_T


def rows(cache: torch.Tensor, table_row: torch.Tensor, pos: torch.Tensor, h: int, scale) -> torch.Tensor:
    """Values [len(pos), D] of the tokens at `pos` in float64.  scale: a number, or (kv_scales, 0 or 1)."""
    pblk = cache.shape[1]
    blk, slot = table_row.long()[pos // pblk], pos % pblk
    x = cache[blk, slot, h]
    x = x.double() if cache.dtype == torch.bfloat16 else _E4M3_T[_as_u8(x).long()]
    if isinstance(scale, tuple):
        e = scale[0][blk, slot // 16, h, scale[1]].double() - 127
        return x * torch.exp2(e)[:, None]
    return x * (1.0 if cache.dtype == torch.bfloat16 else scale)


def visible(p: int, length: int, window: int, sinks: int) -> torch.Tensor:
    t = torch.arange(max(0, min(p + 1, length)))
    return t if window == 0 else t[(t > p - window) | (t < sinks)]


def attention(q, k_cache, v_cache, starts, seq_lens, table, k_scale, v_scale, sm_scale, window=0, sinks=0):
    """(out [T, HQ, D], sum_t w_t |V_t| of the same shape, largest sm_scale * sum_d |q_d K_td| per row [T, HQ])."""
    T, HQ, D = q.shape
    HKV = k_cache.shape[2]
    out = torch.zeros(T, HQ, D, dtype=torch.float64)
    mass, reach = torch.zeros_like(out), torch.zeros(T, HQ, dtype=torch.float64)
    for s in range(table.shape[0]):
        a, b, length = int(starts[s]), int(starts[s + 1]), int(seq_lens[s])
        for row in range(a, b):
            p = length - (b - a) + row - a
            pos = visible(p, length, window, sinks)
            if pos.numel() == 0:
                continue
            for h in range(HKV):
                k = rows(k_cache, table[s], pos, h, k_scale)
                v = rows(v_cache, table[s], pos, h, v_scale)
                heads = slice(h * HQ // HKV, (h + 1) * HQ // HKV)
                x = q[row, heads].double()
                w = torch.softmax(x @ k.T * sm_scale, -1)
                out[row, heads] = w @ v
                mass[row, heads] = w @ v.abs()
                reach[row, heads] = (x.abs() @ k.abs().T).amax(-1) * abs(sm_scale)
    return out, mass, reach
