"""Inputs of the rotating append's tests."""

from __future__ import annotations

import random

import torch

from mini_vllm import torch_path


def append_case(plan, *, dtype, kv_dtype=None, hq=4, hk=2, d=64, page=16, padded=0, seed=0,
                fused=False, position_dtype=torch.int64, size=1.0, max_positions=None):
    """(arguments, pools) of rope_kv_write for sequences of (tokens held, tokens new), on the CPU.
    The pages of the held tokens hold values (and power-of-two scales) already."""
    kv_dtype = kv_dtype or dtype
    g = torch.Generator().manual_seed(seed)
    pages = [range(p // page, -(-(p + n) // page)) for p, n in plan]
    order = list(range(sum(map(len, pages)) + 2))
    random.Random(seed).shuffle(order)
    slots, positions, at = [], [], 0
    for (p, n), held in zip(plan, pages):
        slots += [order[at + j // page - held.start] * page + j % page for j in range(p, p + n)]
        positions += range(p, p + n)
        at += len(held)
    slots += [-1] * padded
    positions += [0] * padded
    t = len(slots)
    x = (torch.randn((t, (hq + 2 * hk) * d), generator=g) * size).to(dtype)
    q, k, v = x.split([hq * d, hk * d, hk * d], dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos, sin = torch_path.rope_tables(d, max_positions or max(positions) + 1, 10000.0)
    pools = {"k_scale": None, "v_scale": None}
    for name in ("key_pool", "value_pool"):
        pool = torch.randn((len(order), page, hk, d), generator=g)
        if kv_dtype == torch.float8_e4m3fn:
            scale = torch.exp2(torch.ceil(torch.log2(pool.abs().amax(dim=(1, 3)) / 448.0)))
            pools[name[0] + "_scale"] = scale
            pool = pool / scale[:, None, :, None]
        pools[name] = pool.to(kv_dtype)
    return {"q": q.view(t, hq, d), "k": k.view(t, hk, d), "v": v.view(t, hk, d),
            "positions": torch.tensor(positions, dtype=position_dtype), "cos": cos, "sin": sin,
            "slot_mapping": torch.tensor(slots, dtype=torch.int32)}, pools


def clone_pools(pools):
    return {k: None if v is None else v.clone() for k, v in pools.items()}


def rotated64(x, c):
    """The rotation in 64 bits, and the size of the two products that it sums."""
    cos, sin = (c[n].double()[c["positions"].long()][:, None] for n in ("cos", "sin"))
    a, b = x.double().chunk(2, dim=-1)
    turned = torch.cat((-b, a), dim=-1)
    return x.double() * cos + turned * sin, (x.double() * cos).abs() + (turned * sin).abs()
