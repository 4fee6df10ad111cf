"""Windowed attention with sinks without a GPU: the oracle's closed forms, the PyTorch path against
it, the refusals of the seam and of the library's plan."""

from __future__ import annotations

import pytest
import torch

from mini_vllm.kernels import extension, ops
from oracle.paged_attention import paged_attention as full_oracle
from oracle.window_attention import window_attention
from window_helpers import assert_close, rolling_batch


def call(batch, **more):
    args = {**batch, **more}
    return ops.paged_window_attention(**args)


def oracle_of(b):
    return window_attention(b["q"], b["key_pool"], b["value_pool"], b["block_tables"],
                            b["cu_seqlens_q"], b["context_lens"], b["window"], b["sinks"],
                            b["scale"], b["k_scale"], b["v_scale"])[0]


def test_a_window_of_one_returns_the_key_itself():
    b = rolling_batch([(40, 7), (1, 1), (33, 1)], 1, 0, hq=4, hk=2, d=32)
    out = oracle_of(b)
    cu = b["cu_seqlens_q"].tolist()
    for s, (ctx, new) in enumerate([(40, 7), (1, 1), (33, 1)]):
        for r in range(new):
            p = ctx - new + r
            v = b["value_pool"][int(b["block_tables"][s, p // 16]), p % 16].double()
            assert torch.equal(out[cu[s] + r], v.repeat_interleave(2, dim=0))


def test_equal_scores_average_the_sinks_and_the_window():
    b = rolling_batch([(100, 1)], 10, 3, hq=2, hk=1, d=32)
    b["q"].zero_()
    keys = [0, 1, 2, *range(90, 100)]
    v = torch.stack([b["value_pool"][int(b["block_tables"][0, j // 16]), j % 16, 0] for j in keys])
    torch.testing.assert_close(oracle_of(b)[0, 1], v.double().mean(0), rtol=0, atol=1e-12)


def test_a_window_past_every_context_is_causal_attention():
    b = rolling_batch([(50, 9), (17, 17), (64, 1)], 64, 0, hq=4, hk=2, d=32)
    full = full_oracle(b["q"], b["key_pool"].nan_to_num(), b["value_pool"].nan_to_num(),
                       b["block_tables"], b["cu_seqlens_q"], b["context_lens"], b["scale"])
    assert (oracle_of(b) - full.double()).abs().max() < 1e-5


@pytest.mark.parametrize("kv_dtype", [torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (16, 4), (33, 17), (1000, 0), (3, 1000)])
def test_torch_path_matches_the_oracle(window, sinks, kv_dtype):
    b = rolling_batch([(40, 7), (1, 1), (33, 1), (0, 1), (5, 0), (70, 70)], window, sinks, hq=4,
                      hk=2, d=32, kv_dtype=kv_dtype)
    assert_close(call(b), b, "torch path")
    # a kernel call on CPU tensors runs the same path, and strictly refuses
    assert torch.equal(call(b, use_cuda=True), call(b))
    with ops.strict_kernels(), pytest.raises(RuntimeError, match="device tensors"):
        call(b, use_cuda=True)


def test_refusals_of_the_seam():
    b = rolling_batch([(80, 7)], 8, 2, hq=4, hk=2, d=32)
    for bad in ({"window": 0}, {"window": -3}, {"sinks": -1}):
        with pytest.raises(ValueError, match="window must be >= 1 and sinks >= 0"):
            call(b, **bad)
    with pytest.raises(ValueError, match="page its table does not hold"):
        call(b, window=60)      # asks for freed pages
    with pytest.raises(ValueError, match="computes"):
        call(b, context_lens=torch.tensor([5], dtype=torch.int32))


@pytest.fixture(scope="module")
def lib():
    return extension.HipExtension(extension.open_library())


def plan(lib, window=128, sinks=4, num_tokens=4, num_seqs=4, max_query_len=1, max_context_len=4096,
         q_dtype=torch.bfloat16, kv_dtype=torch.bfloat16, head_dim=128, options=None):
    return lib.paged_window_attention_plan(num_tokens, num_seqs, 16, 8, head_dim, 16, max_query_len,
                                           max_context_len, window, sinks, q_dtype, kv_dtype, options)


def test_plan_refusals(lib):
    for bad in ({"window": 0}, {"sinks": -1}):
        with pytest.raises(RuntimeError, match="window must be >= 1"):
            plan(lib, **bad)
    with pytest.raises(RuntimeError, match="not served"):
        plan(lib, max_context_len=2**30)
    with pytest.raises(RuntimeError, match="at least max_query_len"):
        plan(lib, num_tokens=10, num_seqs=1, max_query_len=10, max_context_len=9)
    with pytest.raises(RuntimeError, match="head dim"):
        plan(lib, head_dim=96)


def test_decode_schedules(lib):
    """A workgroup per list where that is the faster one, without a workspace; the stream for few
    long lists and for many over fp8; a forced one; none of it for calls without a window."""
    def mode(n, window, **more):
        return plan(lib, window=window, num_tokens=n, num_seqs=n, max_context_len=30000, **more)["decode_mode"]
    fp8 = {"kv_dtype": torch.float8_e4m3fn}
    assert mode(1, 128) == mode(28, 700) == mode(28, 700, **fp8) == mode(300, 4000) == "direct"
    assert mode(1, 4000) == mode(4, 4000, **fp8) == mode(256, 4000, **fp8) == mode(300, 100, **fp8) == "stream"
    assert mode(4200, 100) == "direct" and mode(4200, 100, **fp8) == "grid"
    direct = plan(lib, window=128, options={"decode_schedule": 4})
    assert direct["decode_mode"] == "direct" and direct["workspace_bytes"] == 0
    assert direct["decode_workgroups"] == 4 * 8
    with pytest.raises(RuntimeError, match="out of range"):
        lib.paged_attention_plan(4, 4, 16, 8, 128, 16, 1, 100, torch.bfloat16, torch.bfloat16,
                                 {"decode_schedule": 4})


def test_decode_rows_beside_the_prefill(lib):
    """In the prefill's launch where their lists end within it; a launch of their own for long lists,
    many of them, or shapes that the pair kernel does not take."""
    def mode(n, tokens, window, chunk=512, **more):
        return plan(lib, window=window, num_tokens=n + tokens, num_seqs=n + tokens // chunk,
                    max_query_len=chunk, max_context_len=30000, **more)["decode_mode"]
    fp8 = {"kv_dtype": torch.float8_e4m3fn}
    assert mode(8, 512, 1024) == mode(8, 512, 1024, **fp8) == mode(62, 512, 1024) == "beside"
    assert mode(100, 2048, 1024) == mode(1, 64, 1024, 64, **fp8) == mode(30, 2048, 2000) == "beside"
    assert {mode(1, 64, 1024, 64), mode(31, 512, 4096), mode(250, 4096, 512), mode(16, 512, 2000),
            mode(126, 4096, 1000, **fp8), mode(8, 512, 1024, head_dim=64)} <= {"direct", "stream"}
    assert mode(8, 512, 1024, options={"decode_schedule": 4}) == "direct"
    assert mode(31, 512, 4096, options={"decode_schedule": 5}) == "beside"
    assert mode(8, 512, 1024, head_dim=64, options={"decode_schedule": 5}) in ("direct", "stream")
    beside = plan(lib, window=256, num_tokens=520, num_seqs=9, max_query_len=512)
    assert beside["decode_workgroups"] == 9 * 8
    assert plan(lib, window=256, num_tokens=1024, num_seqs=2, max_query_len=512)["decode_mode"] == "none"
    with pytest.raises(RuntimeError, match="out of range"):
        plan(lib, options={"decode_schedule": 6})
    with pytest.raises(RuntimeError, match="out of range"):
        plan(lib, options={"decode_schedule": 3})


def test_a_plan_goes_by_the_window_not_the_context(lib):
    # the fewest keys of a share at this type are 16: no more workgroups than shares of the window
    stream = {"decode_schedule": 1}
    assert plan(lib, window=128, sinks=4, num_tokens=1, num_seqs=1, max_context_len=2**29,
                options=stream)["decode_workgroups"] == 9
    assert (plan(lib, window=2**31 - 1, sinks=2**31 - 1, options=stream)["decode_workgroups"]
            == lib.paged_attention_plan(4, 4, 16, 8, 128, 16, 1, 4096, torch.bfloat16,
                                        torch.bfloat16)["decode_workgroups"])
    by_row = plan(lib, num_tokens=100, num_seqs=1, max_query_len=100, q_dtype=torch.float32,
                  kv_dtype=torch.float32)
    assert by_row["decode_mode"] == "by_row" and by_row["split_tokens"] >= 64
