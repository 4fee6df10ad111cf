"""Batches of a rolling cache for the windowed attention's tests, and its error bound."""

from __future__ import annotations

import random

import torch

from oracle.window_attention import window_attention


def rolling_batch(pairs, window, sinks, *, dtype=torch.float32, kv_dtype=None, hq=16, hk=8, d=128,
                  page=16, seed=0, spare_rows=0, scale=None, pow2_scales=True):
    """A call of paged_window_attention over sequences of (context, queries), as a dict of its
    arguments on the CPU. Pages that no query sees are freed (table entries -1), and every row of
    the pool that no query sees holds NaN."""
    kv_dtype = kv_dtype or dtype
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    seen, held = [], []
    for s, l in pairs:
        keys = [j for j in range(s) if l > 0 and (j < sinks or j > s - l - window)]
        seen.append(keys)
        held.append(sorted({j // page for j in keys}))
    total = sum(map(len, held)) + 3
    order = list(range(total))
    rng.shuffle(order)
    width = max([-(-s // page) for s, _ in pairs] + [1])
    tables = torch.full((len(pairs), width), -1, dtype=torch.int32)
    live = torch.zeros(total * page, dtype=torch.bool)
    at = 0
    for i, pages in enumerate(held):
        for n in pages:
            tables[i, n] = order[at]
            at += 1
        for j in seen[i]:
            live[int(tables[i, j // page]) * page + j % page] = True
    shape = (total, page, hk, d)
    live = live.view(total, page, 1, 1)
    out = {}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g)
        scales = None
        if kv_dtype == torch.float8_e4m3fn:
            scales = x.abs().amax(dim=(1, 3)) / 448.0
            if pow2_scales:
                scales = torch.exp2(torch.ceil(torch.log2(scales)))
            x = x / scales[:, None, :, None]
        out[name + "_scale"] = scales
        pool = x.to(kv_dtype)
        poison = torch.full(shape, float("nan")).to(kv_dtype)
        out[name] = torch.where(live, pool.float(), poison.float()).to(kv_dtype)
    new = [l for _, l in pairs]
    rows = sum(new) + spare_rows
    cu = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
    return {"q": torch.randn((rows, hq, d), generator=g).to(dtype), "key_pool": out["k"],
            "value_pool": out["v"], "block_tables": tables, "cu_seqlens_q": cu,
            "context_lens": torch.tensor([s for s, _ in pairs], dtype=torch.int32),
            "seq_lens": torch.tensor(new, dtype=torch.int32),
            "max_query_len": max(new + [1]), "max_context_len": max([s for s, _ in pairs] + new + [1]),
            "window": window, "sinks": sinks, "scale": d ** -0.5 if scale is None else scale,
            "k_scale": out["k_scale"], "v_scale": out["v_scale"]}


def on(batch, device):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in batch.items()}


def expected(batch, chunks_only=False):
    """The oracle's outputs and the most a kernel may be off, element by element (``chunks_only``:
    single queries are computed as chunks of one token).

    The sums are in float32: a score of D terms is off by (D + 2) 2^-24 of their size, and so is
    the exponent by that and by its own rounding (at most 2^-22 of the score's size, log2 e and the
    maximum's multiply-add in), which moves a weight by as much relative to it and, through the
    sum, by as much again; an output of n weighted terms is off by (n + 64) 2^-24 of their size
    (64: a weight's own exponential, rescalings, merges and the division). In 16 bits the output is
    rounded once more; a chunk's rows also have their weights rounded to the query's type (half a
    step each, and in float16 at least 2^-25 of the largest; the sum takes them unrounded) and
    the values of an fp8 page with an odd scale rounded likewise: K's by half a step of each of the
    score's terms."""
    q = batch["q"]
    out, absolute, score = window_attention(
        q, batch["key_pool"], batch["value_pool"], batch["block_tables"], batch["cu_seqlens_q"],
        batch["context_lens"], batch["window"], batch["sinks"], batch["scale"], batch["k_scale"],
        batch["v_scale"])
    n = min(int(batch["max_context_len"]), batch["window"] + batch["sinks"])
    moved = score * ((q.shape[2] + 2) * 2.0**-24 + 2.0**-22)
    half = torch.finfo(q.dtype).eps / 2
    weight = torch.zeros(q.shape[0], dtype=torch.float64)
    if q.dtype != torch.float32:
        cu = batch["cu_seqlens_q"].tolist()
        for s, l in enumerate(batch["seq_lens"].tolist()):
            if l > 1 or chunks_only:
                weight[cu[s]:cu[s + 1]] = half
        if batch["k_scale"] is not None and not torch.equal(
                batch["k_scale"], torch.exp2(torch.round(torch.log2(batch["k_scale"])))):
            moved = moved + score * weight[:, None]
            weight = 2 * weight
    tolerance = absolute * (2 * moved[:, :, None] + weight[:, None, None] + (n + 64) * 2.0**-24)
    if q.dtype == torch.float16:
        tolerance += (weight > 0).double()[:, None, None] * n * 2.0**-25 * 5.0   # (|v| < 5 a row)
        tolerance += 2.0**-25                                            # subnormal outputs
    if q.dtype != torch.float32:
        tolerance += half * (out.abs() + tolerance)
    return out, tolerance + 1e-30


def assert_close(actual, batch, msg="", chunks_only=False):
    out, tolerance = expected(batch, chunks_only)
    rows = int(batch["cu_seqlens_q"][-1])
    got = actual.double().cpu()[:rows]
    assert torch.isfinite(got).all(), f"{msg}: non-finite output"
    off = (got - out[:rows]).abs() / tolerance[:rows]
    assert off.max().item() <= 1.0, f"{msg}: {off.max().item():.2f} times the bound, at " \
        f"{tuple(int(i) for i in torch.nonzero(off == off.max())[0])}"
