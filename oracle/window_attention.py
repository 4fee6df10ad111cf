"""Windowed paged attention with sinks in float64: the definition, query by query.

A query at position p sees the keys j <= p with j > p - window or j < sinks. Returned beside the
outputs: what bounds a kernel's rounding, ``absolute`` (the softmax-weighted mean of |v|, the
size of the terms an output sums) and ``score`` (the largest scale * sum |q_i k_i| of a row's
visible keys, the size of the terms a score sums). Rows that belong to no sequence, and those of
a sequence without keys, are zeros.
"""

from __future__ import annotations

import torch

__all__ = ["window_attention"]


def window_attention(q, key_pool, value_pool, block_tables, cu_seqlens_q, context_lens, window,
                     sinks, scale, k_scale=None, v_scale=None):
    q64 = q.double().cpu()
    kp, vp = key_pool.cpu(), value_pool.cpu()
    tables, cu = block_tables.cpu().tolist(), cu_seqlens_q.tolist()
    page_rows, hk = key_pool.shape[1:3]
    hq, d = q.shape[1:]
    out = torch.zeros(q64.shape, dtype=torch.float64)
    absolute = torch.zeros(q64.shape, dtype=torch.float64)
    score = torch.zeros(q64.shape[:2], dtype=torch.float64)
    for s, held in enumerate(context_lens.tolist()):
        rows = range(cu[s], cu[s + 1])
        for r, row in enumerate(rows):
            p = held - len(rows) + r
            keys = [j for j in range(max(p + 1, 0)) if j > p - window or j < sinks]
            if not keys:
                continue
            pages = torch.tensor([tables[s][j // page_rows] for j in keys])
            at = torch.tensor([j % page_rows for j in keys])
            assert int(pages.min()) >= 0, "a visible key without a page"
            k, v = kp[pages, at].double(), vp[pages, at].double()       # V x H_k x D
            if k_scale is not None:
                k = k * k_scale.cpu().double()[pages][:, :, None]
                v = v * v_scale.cpu().double()[pages][:, :, None]
            k = k.repeat_interleave(hq // hk, dim=1)
            v = v.repeat_interleave(hq // hk, dim=1)
            w = torch.softmax((k * q64[row]).sum(-1) * scale, dim=0)    # V x H_q
            out[row] = (w[:, :, None] * v).sum(0)
            absolute[row] = (w[:, :, None] * v.abs()).sum(0)
            score[row] = (k * q64[row]).abs().sum(-1).max(dim=0).values * abs(scale)
    return out, absolute, score
