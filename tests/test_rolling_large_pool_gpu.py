"""The rolling cache's ops over pools whose byte offsets pass 32 bits: what the same pages give at the
start of a small pool, bit for bit."""

from __future__ import annotations

import pytest
import torch

from mini_vllm.kernels import ops
from window_helpers import on, rolling_batch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def bits(pool):
    return pool.view(torch.uint8 if pool.dtype == FP8 else torch.int16)


def far(pool, pages):
    """A pool of `pages` pages whose last ones are `pool`'s, the others NaN."""
    out = torch.empty((pages, *pool.shape[1:]), dtype=pool.dtype, device=pool.device)
    bits(out).fill_(0x7F if pool.dtype == FP8 else 0x7FC0)
    bits(out)[-pool.shape[0]:] = bits(pool)
    return out


def far_pages(pool):
    page_bytes = pool[0].numel() * pool.element_size()
    return (2**32 + 2**30) // page_bytes + pool.shape[0]


@pytest.mark.parametrize("kv_dtype", [torch.bfloat16, FP8])
@pytest.mark.parametrize("d,hq,hk,pairs", [
    (128, 4, 2, [(500, 1), (3, 1), (90, 1)]),                  # decode
    (128, 4, 2, [(300, 130), (64, 64)]),                       # the pair kernel
    (128, 4, 2, [(300, 130), (90, 1), (64, 64), (1, 1)]),      # with decode rows beside
    (128, 3, 3, [(300, 130), (90, 1)]),                        # odd groups
    (64, 4, 2, [(300, 130), (90, 1)]),                         # the general kernel
])
def test_window_attention(device, kv_dtype, d, hq, hk, pairs):
    b = on(rolling_batch(pairs, 60, 5, dtype=torch.bfloat16, kv_dtype=kv_dtype, hq=hq, hk=hk, d=d), device)
    want = ops.paged_window_attention(**b, use_cuda=True)
    assert torch.isfinite(want.float()).all()
    pages = far_pages(b["key_pool"])
    shift = pages - b["key_pool"].shape[0]
    for n in ("key_pool", "value_pool"):
        b[n] = far(b[n], pages)
    for n in ("k_scale", "v_scale"):
        if b[n] is not None:
            b[n] = torch.cat([torch.ones(shift, hk, device=device), b[n]])
    b["block_tables"] = torch.where(b["block_tables"] < 0, -1, b["block_tables"] + shift).to(torch.int32)
    assert torch.equal(ops.paged_window_attention(**b, use_cuda=True), want)


@pytest.mark.parametrize("kv_dtype", [torch.bfloat16, FP8])
def test_rope_write(device, kv_dtype):
    g = torch.Generator().manual_seed(0)
    tokens, hq, hk, d, page, blocks = 50, 4, 2, 128, 16, 6
    q, k, v = (torch.randn(tokens, h, d, generator=g).to(torch.bfloat16).to(device) for h in (hq, hk, hk))
    angle = torch.rand(100, d, generator=g) * 6
    tables = [f(angle).to(device) for f in (torch.cos, torch.sin)]
    positions = torch.arange(tokens, dtype=torch.int32, device=device)
    slots = torch.arange(tokens, dtype=torch.int32, device=device) + page
    pools = [torch.zeros((blocks, page, hk, d), device=device).to(kv_dtype) for _ in range(2)]
    scales = {}
    if kv_dtype == FP8:
        scales = {n: torch.zeros(blocks, hk, device=device) for n in ("k_scale", "v_scale")}
    large = [far(x, far_pages(x)) for x in pools]
    shift = large[0].shape[0] - blocks
    large_scales = {n: torch.zeros(shift + blocks, hk, device=device) for n in scales}
    args = (q, k, v, positions, *tables)
    want = ops.rope_kv_write(*args, *pools, slots, use_cuda=True, **scales)
    got = ops.rope_kv_write(*args, *large, slots + shift * page, use_cuda=True, **large_scales)
    assert torch.equal(got, want)
    for a, b in zip(large, pools):
        assert torch.equal(bits(a[-blocks:]), bits(b))
        assert (bits(a[:-blocks]) == (0x7F if kv_dtype == FP8 else 0x7FC0)).all()
    for n in scales:
        assert torch.equal(large_scales[n][-blocks:], scales[n]) and not large_scales[n][:-blocks].any()
