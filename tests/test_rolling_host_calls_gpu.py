"""The native bodies of the rolling cache's ops against their Python ones: the same bits where they
serve a call, None where a call is not exactly what the kernels take."""

from __future__ import annotations

import pytest
import torch

from mini_vllm.kernels import extension as ext_module
from mini_vllm.kernels import ops
from rope_write_helpers import append_case, clone_pools
from window_helpers import on, rolling_batch

FP8 = torch.float8_e4m3fn


def test_the_bodies_leave_host_tensors_alone():
    host = ext_module.open_host()
    if host is None:
        pytest.skip("the host module is not built")
    entries = host.rolling_entries(*[0] * 4)
    x = torch.zeros(2, 64)
    assert host.paged_window_attention(entries, {}, *[x] * 14) is None
    assert host.rope_kv_write(entries, *[x] * 11) is None
    for wrong in (x, host.entries(*[0] * 7)):
        with pytest.raises(ValueError):
            host.paged_window_attention(wrong, {}, *[x] * 14)
        with pytest.raises(ValueError):
            host.rope_kv_write(wrong, *[x] * 11)


def python_body(extension, call):
    host, extension._host = extension._host, None
    try:
        return call()
    finally:
        extension._host = host


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [[(300, 1), (17, 1)], [(200, 64), (70, 1)]])
@pytest.mark.parametrize("dtype,kv", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, FP8)])
def test_window_attention(extension, device, pairs, dtype, kv):
    b = on(rolling_batch(pairs, 50, 4, dtype=dtype, kv_dtype=kv), device)

    def call(**more):
        return ops.paged_window_attention(**{**b, **more}, use_cuda=True)
    want = python_body(extension, call)
    args = [b[n] for n in ("q", "key_pool", "value_pool", "block_tables", "cu_seqlens_q",
                           "context_lens", "seq_lens", "max_query_len", "max_context_len", "window",
                           "sinks", "scale", "k_scale", "v_scale")]
    own = extension.try_paged_window_attention(*args)
    assert own is not None and torch.equal(own, want) and torch.equal(call(), want)
    for i, other in ((0, b["q"][:, :-1]), (0, b["q"].double()), (3, b["block_tables"].long()),
                     (5, b["context_lens"].cpu()), (7, True), (9, 0), (9, 2**31), (9, 50.0), (10, -1),
                     (11, 1), (1, b["key_pool"][:-1])):
        assert extension.try_paged_window_attention(*args[:i], other, *args[i + 1:]) is None
    wide = on(rolling_batch(pairs, 2**40, 4, dtype=dtype, kv_dtype=kv), device)
    assert torch.equal(call(**wide), python_body(extension, lambda: call(**wide)))
    with extension.recording_workspaces() as held:      # the buffers that a graph keeps alive
        assert extension.try_paged_window_attention(*args) is None
        assert torch.equal(call(), want)
    need = extension.paged_window_attention_plan(
        b["q"].shape[0], len(pairs), 16, 8, 128, 16, b["max_query_len"], b["max_context_len"], 50, 4,
        dtype, kv or dtype)["workspace_bytes"]
    assert bool(held) == (need > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("plan", [[(37, 1)], [(5, 20), (0, 33)]])
@pytest.mark.parametrize("dtype,kv", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, FP8)])
def test_rope_write(extension, device, plan, dtype, kv):
    c, pools = append_case(plan, dtype=dtype, kv_dtype=kv, padded=2)
    c = {n: x.to(device) for n, x in c.items()}
    pools = {n: None if x is None else x.to(device) for n, x in pools.items()}
    want = clone_pools(pools)
    q = python_body(extension, lambda: ops.rope_kv_write(**c, **want, use_cuda=True))
    got = clone_pools(pools)
    args = [{**c, **got}[n] for n in ("q", "k", "v", "positions", "cos", "sin", "key_pool",
                                      "value_pool", "slot_mapping", "k_scale", "v_scale")]
    own = extension.try_rope_kv_write(*args)
    assert own is not None and torch.equal(own, q)
    for n, x in want.items():
        assert x is None or torch.equal(got[n].view(torch.uint8), x.view(torch.uint8))
    for i, other in ((0, c["q"][:, :, :-16]), (1, c["k"].double()), (2, c["v"][:-1]),
                     (3, c["positions"].float()), (4, c["cos"].half()), (5, c["sin"][:, :-1]),
                     (6, pools["key_pool"][:-1]), (8, c["slot_mapping"].long()),
                     (8, c["slot_mapping"].cpu()), (9, c["cos"])):
        assert extension.try_rope_kv_write(*args[:i], other, *args[i + 1:]) is None
    for n, x in want.items():     # a call that is not served has done nothing
        assert x is None or torch.equal(got[n].view(torch.uint8), x.view(torch.uint8))
