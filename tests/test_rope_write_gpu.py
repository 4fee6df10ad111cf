"""The rotating append on the GPU: bit for bit rope then the write for pools of the inputs' type,
and bit for bit the PyTorch path's codes and scales (itself held to 64 bits) for fp8 pools."""

from __future__ import annotations

import pytest
import torch

from mini_vllm import torch_path
from mini_vllm.kernels import ops
from rope_write_helpers import append_case, clone_pools, rotated64

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
PLANS = {"one": [(37, 1)], "decode": [(17 * i % 90, 1) for i in range(70)],
         "ragged": [(5, 20), (0, 1), (16, 16), (40, 3), (31, 2), (0, 100), (63, 65)],
         "large": [(7, 1500), (0, 600), (33, 1), (100, 77)],
         "many": [(i % 50, 1) for i in range(2100)]}


def to(device, d):
    """On the device, column views staying views of one tensor."""
    if d.get("q") is not None and not d["q"].is_contiguous():
        t, hq, dim = d["q"].shape
        hk = d["k"].shape[1]
        x = d["q"]._base.to(device)
        q, k, v = x.split([hq * dim, hk * dim, hk * dim], dim=1)
        rest = {n: x.to(device) for n, x in d.items() if n not in "qkv"}
        return {**rest, "q": q.view(t, hq, dim), "k": k.view(t, hk, dim), "v": v.view(t, hk, dim)}
    return {n: None if x is None else x.to(device) for n, x in d.items()}


def bits(x):
    """Codes, the two of NaN (whose sign no arithmetic defines) as one."""
    if x.dtype != FP8:
        return x
    code = x.view(torch.uint8)
    return torch.where((code & 0x7F) == 0x7F, 0x7F, code)


def check(device, c, pools):
    """The kernel's q and pools against the PyTorch path's on the CPU."""
    want = clone_pools(pools)
    want_q = ops.rope_kv_write(**c, **want)
    got = to(device, pools)
    got_q = ops.rope_kv_write(**to(device, c), **got, use_cuda=True)
    assert torch.equal(got_q.cpu(), want_q)
    for name, x in want.items():
        if x is not None:
            assert torch.equal(bits(got[name].cpu()), bits(x)), name
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("kv", ["same", "fp8"])
def test_append(device, plan, dtype, kv):
    c, pools = append_case(PLANS[plan], dtype=dtype, kv_dtype=FP8 if kv == "fp8" else None,
                           padded=3, fused=plan != "ragged", hq=4, hk=2, d=64)
    check(device, c, pools)


@pytest.mark.parametrize("hq,hk,d,page", [(16, 8, 128, 16), (3, 1, 32, 4), (5, 5, 256, 64),
                                          (2, 1, 128, 1), (8, 2, 64, 128), (7, 7, 32, 32)])
@pytest.mark.parametrize("kv", ["same", "fp8"])
@pytest.mark.parametrize("position_dtype", [torch.int32, torch.int64])
def test_layouts(device, hq, hk, d, page, kv, position_dtype):
    c, pools = append_case(PLANS["ragged"], dtype=torch.bfloat16, kv_dtype=FP8 if kv == "fp8" else None,
                           hq=hq, hk=hk, d=d, page=page, position_dtype=position_dtype, fused=True)
    check(device, c, pools)


@pytest.mark.parametrize("d", [16, 48, 96, 1024])
def test_head_dims_of_same_type_pools(device, d):
    c, pools = append_case(PLANS["ragged"], dtype=torch.float16, hq=3, hk=1, d=d)
    check(device, c, pools)


def test_against_64_bits(device):
    c, pools = append_case(PLANS["large"], dtype=torch.bfloat16, hq=8, hk=4, d=128)
    got = to(device, pools)
    q = ops.rope_kv_write(**to(device, c), **got, use_cuda=True).cpu().double()
    k = got["key_pool"].cpu().view(-1, 4, 128)[c["slot_mapping"].long()].double()
    for y, x in ((q, c["q"]), (k, c["k"])):
        want, size = rotated64(x, c)
        assert ((y - want).abs() <= size * 3 * 2.0**-24 + 2.0**-8 * (want.abs() + size * 2.0**-22)).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("large", [False, True])
def test_a_page_whose_scale_grows_step_by_step(device, page, large):
    """One token a step into one page (beside others), each larger than the last; then the page
    is opened again. The many-token form too, its other rows padding."""
    pools = wanted = None
    for step in range(20):
        c, fresh = append_case([(step % page, 1), (3, 1)], dtype=torch.float32, kv_dtype=FP8, page=page,
                               hq=2, hk=2, d=32, seed=1, padded=2046 if large else 0)
        for n in "kv":
            c[n] = c[n] * 1.7**step * (1 + torch.arange(2)[None, :, None])
        c["slot_mapping"][0] = 2 * page + step % page
        c["slot_mapping"][1] = 3
        pools, wanted = (pools, wanted) if pools else (to(device, fresh), fresh)
        ops.rope_kv_write(**c, **wanted)
        ops.rope_kv_write(**to(device, c), **pools, use_cuda=True)
        for name, x in wanted.items():
            assert torch.equal(bits(pools[name].cpu()), bits(x)), (step, name)


def test_positions_slots_and_values_out_of_range(device):
    c, pools = append_case(PLANS["ragged"], dtype=torch.bfloat16, hq=4, hk=2, d=64)
    before = clone_pools(pools)
    c["positions"][3], c["positions"][5] = -1, 10**12
    c["slot_mapping"][7] = 2**31 - 1
    got = to(device, pools)
    q = ops.rope_kv_write(**to(device, c), **got, use_cuda=True).cpu()
    assert q[[3, 5]].isnan().all() and q[[0, 1, 2, 4, 6, 7]].isfinite().all()
    keys = got["key_pool"].cpu().view(-1, 2, 64)
    assert keys[c["slot_mapping"][[3, 5]].long()].isnan().all()
    written = c["slot_mapping"].long()
    rest = torch.ones(keys.shape[0], dtype=torch.bool)
    rest[written[written < keys.shape[0]]] = False
    assert torch.equal(keys[rest], before["key_pool"].view(-1, 2, 64)[rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fp8_values_that_are_not_finite_or_zero(device, dtype):
    c, pools = append_case(PLANS["ragged"], dtype=dtype, kv_dtype=FP8, hq=4, hk=2, d=64)
    c["v"][3, 1, 7], c["v"][4, 0, 9], c["v"][5, 0, 0] = float("inf"), float("nan"), float("-inf")
    c["k"][8, 1, 40] = float("nan")
    c["v"][21:37] = 0.0     # a whole page of zeros
    c["v"][50, 0], c["v"][60] = 3e38, 1e-38
    check(device, c, pools)


def test_refusals(device, extension):
    c, pools = append_case(PLANS["ragged"], dtype=torch.bfloat16, hq=4, hk=2, d=64)
    c, pools = to(device, c), to(device, pools)

    def refused(words, **more):
        with pytest.raises(RuntimeError, match=words):
            ops.rope_kv_write(**{**c, **pools, **more}, use_cuda=True)
    refused("share", k=c["k"].float(), v=c["v"].float(), key_pool=pools["key_pool"].float(),
            value_pool=pools["value_pool"].float())
    refused("T x H_q", k=c["k"][:-1], v=c["v"][:-1])
    refused("pool", key_pool=pools["key_pool"].half(), value_pool=pools["value_pool"].half())
    refused("num_blocks x P x 2 x 64", key_pool=pools["key_pool"][..., :32].contiguous(),
            value_pool=pools["value_pool"][..., :32].contiguous())
    refused("contiguous", key_pool=pools["key_pool"].transpose(0, 1))
    refused("positions", positions=c["positions"][:-1])
    refused("slot_mapping", slot_mapping=c["slot_mapping"].long())
    refused("tables", cos=c["cos"][:, :32], sin=c["sin"][:, :32])
    refused("float32", cos=c["cos"].double(), sin=c["sin"].double())
    refused("only to a float8", k_scale=torch.ones(1, device=device), v_scale=torch.ones(1, device=device))
    fp8 = {n: pools[n].to(FP8) for n in ("key_pool", "value_pool")}
    refused("needs a contiguous float32", **fp8)
    refused("power of two", key_pool=pools["key_pool"][:, :12].contiguous(),
            value_pool=pools["value_pool"][:, :12].contiguous())
    none = {n: c[n][:0] for n in ("q", "k", "v", "positions", "slot_mapping")}
    assert ops.rope_kv_write(**{**c, **none, **pools}, use_cuda=True).shape == (0, 4, 64)


def test_strides_and_alignment(device):
    """Head-major, misaligned and single-token inputs: the same results as contiguous ones."""
    for plan in ("ragged", "one"):
        c, pools = append_case(PLANS[plan], dtype=torch.bfloat16, hq=4, hk=2, d=64)
        c = to(device, c)
        want = to(device, pools)
        want_q = ops.rope_kv_write(**c, **want, use_cuda=True)
        for name in ("heads", "odd", "wide"):
            d = dict(c)
            for n in "qkv":
                x = c[n]
                if name == "heads":
                    d[n] = x.transpose(0, 1).contiguous().transpose(0, 1)
                elif name == "odd":
                    d[n] = torch.empty(x.numel() + 1, dtype=x.dtype, device=device)[1:].view(x.shape)
                    d[n].copy_(x)
                else:
                    d[n] = torch.empty((x.shape[0], x.shape[1], 67), dtype=x.dtype, device=device)[..., 1:65]
                    d[n].copy_(x)
            got = to(device, pools)
            assert torch.equal(ops.rope_kv_write(**d, **got, use_cuda=True), want_q)
            assert torch.equal(got["key_pool"], want["key_pool"])
            assert torch.equal(got["value_pool"], want["value_pool"])


@pytest.mark.parametrize("kv", ["same", "fp8"])
def test_captured_and_replayed(device, kv):
    c, pools = append_case(PLANS["decode"], dtype=torch.bfloat16, kv_dtype=FP8 if kv == "fp8" else None,
                           hq=4, hk=2, d=64)
    c = to(device, c)
    got = to(device, pools)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        q = ops.rope_kv_write(**c, **got, use_cuda=True)
    for _ in range(3):
        for n, x in pools.items():
            if x is not None:
                got[n].copy_(x)
        c["q"].mul_(-1.5)
        c["v"].mul_(-1.5)
        want = to(device, pools)
        graph.replay()
        want_q = ops.rope_kv_write(**c, **want, use_cuda=True)
        torch.cuda.synchronize()
        assert torch.equal(q, want_q)
        for n, x in want.items():
            if x is not None:
                assert torch.equal(bits(got[n]), bits(x))


@pytest.mark.parametrize("kv", ["same", "fp8"])
def test_append_then_windowed_attention(device, kv):
    """A rolling cache as a server runs it: chunks, then single tokens, the pages behind the window
    handed out again; the attention over what the appends left against the oracle on the same pool."""
    from window_helpers import assert_close

    window, sinks, page, hq, hk, d = 40, 5, 16, 4, 2, 128
    kv_dtype = FP8 if kv == "fp8" else torch.bfloat16
    g = torch.Generator().manual_seed(3)
    cos, sin = torch_path.rope_tables(d, 600, 10000.0, device=device)
    blocks = 24
    shape = (blocks, page, hk, d)
    k_pool, v_pool = (torch.zeros(shape, device=device).to(kv_dtype) for _ in range(2))
    scales = [torch.zeros(blocks, hk, device=device) if kv == "fp8" else None for _ in range(2)]
    free, held = list(range(blocks)), [{}, {}]
    lengths, table_width = [0, 0], 40
    for step in range(14):
        new = [90, 33] if step == 0 else [50, 1] if step == 3 else [1, 1]
        tables = torch.full((2, table_width), -1, dtype=torch.int32)
        slots, positions = [], []
        for s in range(2):
            start, end = lengths[s], lengths[s] + new[s]
            for n in [n for n in held[s] if n >= -(-sinks // page) and (n + 1) * page <= start - window + 1]:
                free.append(held[s].pop(n))
            for n in range(start // page, -(-end // page)):
                if n not in held[s]:
                    held[s][n] = free.pop(0)
            for n, b in held[s].items():
                tables[s, n] = b
            slots += [held[s][j // page] * page + j % page for j in range(start, end)]
            positions += range(start, end)
            lengths[s] = end
        t = len(slots)
        q, k, v = (torch.randn((t, h, d), generator=g).to(torch.bfloat16).to(device) for h in (hq, hk, hk))
        q = ops.rope_kv_write(q, k, v, torch.tensor(positions, device=device), cos, sin, k_pool, v_pool,
                              torch.tensor(slots, dtype=torch.int32, device=device), use_cuda=True,
                              k_scale=scales[0], v_scale=scales[1])
        batch = {"q": q, "key_pool": k_pool, "value_pool": v_pool, "block_tables": tables.to(device),
                 "cu_seqlens_q": torch.tensor([0, new[0], t], dtype=torch.int32, device=device),
                 "context_lens": torch.tensor(lengths, dtype=torch.int32, device=device),
                 "seq_lens": torch.tensor(new, dtype=torch.int32, device=device),
                 "max_query_len": max(new), "max_context_len": max(lengths), "window": window,
                 "sinks": sinks, "scale": d ** -0.5, "k_scale": scales[0], "v_scale": scales[1]}
        out = ops.paged_window_attention(**batch, use_cuda=True)
        cpu = {n: x.cpu() if isinstance(x, torch.Tensor) else x for n, x in batch.items()}
        assert_close(out, cpu, f"step {step}")
