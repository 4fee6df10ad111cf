"""Windowed attention with sinks on the GPU against the float64 oracle: every kernel behind it, at
the lengths, windows, sinks and layouts where their edges meet. Pages that no query sees are
freed in every batch, and the rows of held pages that no query sees hold NaN."""

from __future__ import annotations

import pytest
import torch

from mini_vllm.kernels import ops
from window_helpers import assert_close, expected, on, rolling_batch

pytestmark = pytest.mark.gpu

DECODES = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (64, 1), (100, 1), (333, 1), (1000, 1)]
CHUNKS = [(5, 5), (64, 64), (65, 65), (200, 33), (300, 2), (700, 300), (130, 129)]
MIXED = [(90, 1), (200, 33), (0, 1), (64, 64), (7, 0), (500, 1), (130, 2), (1, 1)]
WINDOWS = [(1, 0), (1, 1), (7, 4), (16, 16), (17, 0), (63, 17), (64, 64), (100, 1), (333, 5),
           (5000, 3), (2, 400), (2**40, 2**40)]
TYPES = [(torch.float32, None), (torch.float16, None), (torch.bfloat16, None),
         (torch.float32, torch.float8_e4m3fn), (torch.bfloat16, torch.float8_e4m3fn),
         (torch.float16, torch.float8_e4m3fn)]


def call(batch, device, **more):
    args = {**on(batch, device), **more}
    return ops.paged_window_attention(**args, use_cuda=True)


@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_decode(device, window, sinks, dtype, kv_dtype):
    b = rolling_batch(DECODES, window, sinks, dtype=dtype, kv_dtype=kv_dtype)
    assert_close(call(b, device), b, f"{window} {sinks}")


@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_prefill(device, window, sinks, dtype, kv_dtype):
    b = rolling_batch(CHUNKS, window, sinks, dtype=dtype, kv_dtype=kv_dtype, hq=4, hk=2)
    assert_close(call(b, device), b, f"{window} {sinks}")


LAYOUTS = [(4, 4, 128, 16), (6, 2, 128, 16), (8, 2, 128, 32), (8, 2, 64, 16), (3, 3, 64, 16),
           (4, 2, 256, 16), (2, 2, 32, 16), (12, 2, 32, 4), (4, 2, 128, 1), (4, 2, 128, 8),
           (4, 2, 128, 128), (5, 1, 256, 64)]


@pytest.mark.parametrize("dtype,kv_dtype", [TYPES[0], TYPES[2], TYPES[4]])
@pytest.mark.parametrize("hq,hk,d,page", LAYOUTS)
@pytest.mark.parametrize("window,sinks", [(40, 5), (130, 20)])
def test_layouts(device, hq, hk, d, page, window, sinks, dtype, kv_dtype):
    b = rolling_batch(MIXED, window, sinks, dtype=dtype, kv_dtype=kv_dtype, hq=hq, hk=hk, d=d,
                      page=page, seed=hq * d)
    assert_close(call(b, device), b, f"{hq}/{hk} {d} page {page}")


@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scales(device, dtype, scale):
    b = rolling_batch(MIXED, 50, 3, dtype=dtype, hq=4, hk=2, scale=scale)
    assert_close(call(b, device), b, f"scale {scale}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp8_scales_that_are_no_powers_of_two(device, dtype):
    b = rolling_batch(MIXED + CHUNKS, 90, 9, dtype=dtype, kv_dtype=torch.float8_e4m3fn, hq=4, hk=2,
                      pow2_scales=False)
    assert_close(call(b, device), b)


SCHEDULES = {"stream": 1, "grid": 2, "direct": 4}


@pytest.mark.parametrize("dtype,kv_dtype", TYPES)
@pytest.mark.parametrize("schedule", SCHEDULES)
@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (4, 1, 64), (3, 3, 32), (6, 1, 256)])
def test_decode_schedules(device, extension, schedule, hq, hk, d, dtype, kv_dtype):
    b = rolling_batch(DECODES + [(0, 1), (40, 0)], 70, 9, dtype=dtype, kv_dtype=kv_dtype, hq=hq, hk=hk, d=d)
    args = on(b, device)
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], 1, b["max_context_len"], 70, 9, b["scale"],
        args["k_scale"], args["v_scale"], plan_options={"decode_schedule": SCHEDULES[schedule]})
    assert_close(got, b, schedule)


@pytest.mark.parametrize("schedule", SCHEDULES)
@pytest.mark.parametrize("n", [65, 300])
def test_many_sequences(device, extension, n, schedule):
    """More sequences than a wave has lanes, and rows without keys among them."""
    pairs = [(37 * i % 301, 1) for i in range(n)]
    b = rolling_batch(pairs, 100, 4, dtype=torch.bfloat16, hq=4, hk=2)
    options = {"decode_schedule": SCHEDULES[schedule], "decode_split_tokens": 64}
    args = on(b, device)
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], 1, b["max_context_len"], 100, 4, b["scale"],
        plan_options=options)
    assert_close(got, b, schedule)


def test_many_kv_heads_take_the_grid(device):
    b = rolling_batch(DECODES + [(3000, 1)], 600, 4, dtype=torch.bfloat16, hq=32, hk=32, d=64)
    assert_close(call(b, device), b)


@pytest.mark.parametrize("chunks", [1, 70])
@pytest.mark.parametrize("kv_dtype", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("pieces", [1, 3, 64])
@pytest.mark.parametrize("schedule", [0, 1, 2])
def test_prefill_schedules(device, extension, chunks, kv_dtype, pieces, schedule):
    """The pair kernel's items whole and cut, on the grid and listed, for more sequences than a
    wave has lanes too."""
    pairs = [(900, 150)] + [(20 + 3 * i, 2 + i % 5 if i % 3 else 1) for i in range(chunks - 1)]
    b = rolling_batch(pairs, 400, 7, dtype=torch.bfloat16, kv_dtype=kv_dtype, hq=4, hk=2)
    args = on(b, device)
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], b["max_query_len"], b["max_context_len"], 400, 7,
        b["scale"], args["k_scale"], args["v_scale"],
        plan_options={"prefill_schedule": schedule, "prefill_pieces": pieces,
                      "prefill_share_tiles": 1, "prefill_piece_pct": 50})
    assert_close(got, b)


BESIDE = MIXED + DECODES + [(40, 0), (0, 1)]


@pytest.mark.parametrize("dtype,kv_dtype", [x for x in TYPES if x[0] != torch.float32])
@pytest.mark.parametrize("hq,hk", [(16, 8), (4, 1), (6, 1), (16, 2)])
@pytest.mark.parametrize("schedule,pieces", [(1, 3), (2, 1), (0, 1)])
@pytest.mark.parametrize("n", [1, 5])
def test_decode_rows_beside_the_prefill(device, extension, n, schedule, pieces, hq, hk, dtype, kv_dtype):
    """In the prefill's launch, behind listed items and on the item grid, up to 64 sequences and more."""
    b = rolling_batch(BESIDE * n, 70, 9, dtype=dtype, kv_dtype=kv_dtype, hq=hq, hk=hk, spare_rows=3)
    args = on(b, device)
    options = {"decode_schedule": 5, "prefill_schedule": schedule, "prefill_pieces": pieces}
    plan = extension.paged_window_attention_plan(
        b["q"].shape[0], len(BESIDE) * n, hq, hk, 128, 16, b["max_query_len"], b["max_context_len"], 70, 9,
        b["q"].dtype, b["key_pool"].dtype, options)
    assert plan["decode_mode"] == "beside"
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], b["max_query_len"], b["max_context_len"], 70, 9,
        b["scale"], args["k_scale"], args["v_scale"], plan_options=options)
    assert_close(got, b)


@pytest.mark.parametrize("n", [0, 70])
def test_decode_rows_beside_items_of_128(device, extension, n):
    pairs = [(600 - 7 * i, 512) for i in range(3)] + [(300, 1), (0, 1), (900, 1)] + [(9 + i, 1) for i in range(n)]
    b = rolling_batch(pairs, 200, 5, dtype=torch.bfloat16, kv_dtype=torch.float8_e4m3fn, hq=32, hk=8)
    plan = extension.paged_window_attention_plan(
        b["q"].shape[0], len(pairs), 32, 8, 128, 16, 512, 900, 200, 5, torch.bfloat16, torch.float8_e4m3fn)
    assert (plan["decode_mode"], plan["prefill_item"]) == ("beside", 128)
    assert_close(call(b, device), b)


def test_decode_rows_beside_a_prefill_without_a_positive_scale(device, extension):
    b = rolling_batch(BESIDE, 70, 9, dtype=torch.bfloat16, hq=4, hk=2, scale=-0.2)
    args = on(b, device)
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], b["max_query_len"], b["max_context_len"], 70, 9,
        b["scale"], plan_options={"decode_schedule": 5})
    assert_close(got, b)


@pytest.mark.parametrize("staging", [0, 1])
def test_long_window_of_a_long_context(device, extension, staging):
    b = rolling_batch([(9000, 100), (8200, 1)], 4100, 21, dtype=torch.bfloat16, hq=2, hk=1)
    args = on(b, device)
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], 100, 9000, 4100, 21, b["scale"],
        plan_options={"prefill_staging": staging})
    assert_close(got, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_window_past_every_context_equals_full_attention(device, dtype):
    b = rolling_batch(MIXED[:2] + MIXED[3:4] + MIXED[5:], 10**6, 0, dtype=dtype)
    args = on(b, device)
    full = ops.paged_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], b["max_query_len"], b["max_context_len"], b["scale"],
        use_cuda=True)
    out, tolerance = expected(b)
    assert ((call(b, device) - full).double().cpu().abs() <= 2 * tolerance).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairs", [DECODES, MIXED])
def test_rows_behind_the_last_sequence_stay(device, extension, pairs, dtype):
    b = rolling_batch(pairs, 30, 4, dtype=dtype, hq=4, hk=2, spare_rows=5)
    args = on(b, device)
    out = torch.full_like(args["q"], 7.0)
    got = extension.paged_window_attention(
        args["q"], args["key_pool"], args["value_pool"], args["block_tables"], args["cu_seqlens_q"],
        args["context_lens"], args["seq_lens"], b["max_query_len"], b["max_context_len"], 30, 4,
        b["scale"], out=out)
    assert got is out
    assert_close(out, b)
    assert bool((out[-5:] == 7.0).all())


@pytest.mark.parametrize("hq,hk,d,page", [(4, 2, 128, 16), (3, 1, 128, 16), (4, 2, 64, 16), (4, 2, 128, 8)])
@pytest.mark.parametrize("pairs,spare", [([(90, 2), (50, 1)], 1), ([(90, 2), (0, 1)], 1),
                                         ([(200, 64), (30, 1), (0, 1)], 126),
                                         ([(300, 3)] + [(i, 1) for i in range(70)], 140)])
def test_padded_queries_that_look_like_chunks_only(device, extension, pairs, spare, hq, hk, d, page):
    """q holding rows of no sequence, as many as make its count that of chunks alone."""
    b = rolling_batch(pairs, 30, 4, dtype=torch.bfloat16, hq=hq, hk=hk, d=d, page=page, spare_rows=spare)
    assert b["q"].shape[0] == len(pairs) * b["max_query_len"]
    args = on(b, device)
    for options in (None, {"prefill_schedule": 1, "prefill_share_tiles": 1}):
        out = torch.full_like(args["q"], 7.0)
        extension.paged_window_attention(
            args["q"], args["key_pool"], args["value_pool"], args["block_tables"],
            args["cu_seqlens_q"], args["context_lens"], args["seq_lens"], b["max_query_len"],
            b["max_context_len"], 30, 4, b["scale"], out=out, plan_options=options)
        assert_close(out, b, str(options), chunks_only=True)
        assert bool((out[-spare:] == 7.0).all())


def test_misaligned_queries_and_refusals(device, extension):
    b = on(rolling_batch(MIXED, 30, 4, dtype=torch.bfloat16, hq=4, hk=2), device)
    shifted = torch.empty(b["q"].numel() + 1, dtype=torch.bfloat16, device=device)[1:].view(b["q"].shape)
    shifted.copy_(b["q"])
    assert torch.equal(call(b, device, q=shifted), call(b, device))
    pool = torch.empty(b["key_pool"].numel() + 1, dtype=torch.bfloat16, device=device)[1:].view(
        b["key_pool"].shape)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        call(b, device, key_pool=pool)
    with pytest.raises(RuntimeError, match="float64"):
        call(b, device, q=b["q"].double())
    with pytest.raises(RuntimeError, match="contiguous"):
        call(b, device, q=b["q"].transpose(0, 1))
    with pytest.raises(RuntimeError, match="float8 pool"):
        call(b, device, k_scale=torch.ones(1, device=device), v_scale=torch.ones(1, device=device))
    with pytest.raises(ValueError, match="window must be >= 1"):
        call(b, device, window=0)
    empty = {**b, "q": b["q"][:0], "block_tables": b["block_tables"][:0],
             "cu_seqlens_q": b["cu_seqlens_q"][:1], "context_lens": b["context_lens"][:0],
             "seq_lens": b["seq_lens"][:0]}
    assert call(empty, device).shape == (0, 4, 128)


@pytest.mark.parametrize("pairs", [DECODES, [(900, 150), (64, 64), (90, 1)]])
def test_captured_and_replayed_on_another_stream(device, pairs):
    b = on(rolling_batch(pairs, 100, 4, dtype=torch.bfloat16), device)
    b2 = on(rolling_batch(pairs, 100, 4, dtype=torch.bfloat16, seed=1), device)
    want = [call(b, device).clone(), call({**b, "q": b2["q"]}, device).clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q = b["q"].clone()
    with torch.cuda.stream(side):
        call(b, device, q=q)        # the stream's workspace exists before the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(b, device, q=q)
    for i in (0, 1, 0, 1):
        q.copy_(b["q"] if i == 0 else b2["q"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), f"replay on inputs {i}"
        call(b2, device)            # eager work between the replays
        torch.cuda.synchronize()


def test_two_graphs_and_eager_calls_share_no_workspace(device):
    """Two graphs captured on one stream that has no workspace yet, replayed side by side on two
    streams, then after a larger eager call has grown that stream's workspace."""
    cases = [on(rolling_batch(pairs, 4000, 4, dtype=torch.bfloat16), device)
             for pairs in ([(5000, 1)], [(4500, 1), (900, 200)])]
    large = on(rolling_batch([(5000, 1)] * 3 + [(4000, 500)], 4000, 4, dtype=torch.bfloat16), device)
    want = [call(b, device).clone() for b in cases]
    large_want = call(large, device).clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs = [], []
    for b in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            outs.append(call(b, device))
        graphs.append(graph)
    for round_ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams[1:]):
            with torch.cuda.stream(stream):
                graph.replay()
        if round_ > 0:
            with torch.cuda.stream(streams[0]):
                got = call(large, device)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]), round_
        assert round_ == 0 or torch.equal(got, large_want)


@pytest.mark.parametrize("dtype,kv_dtype", [TYPES[0], TYPES[2], TYPES[4]])
@pytest.mark.parametrize("d", [64, 128])
def test_a_freed_page_that_is_seen_reads_within_the_pool(device, d, dtype, kv_dtype):
    """A window larger than the one pages were freed for: the sequences it makes no difference to
    are right, the others' rows are whatever the pool's last page gives."""
    b = rolling_batch(MIXED, 40, 5, dtype=dtype, kv_dtype=kv_dtype, hq=4, hk=2, d=d)
    out = call({**b, "window": 4000}, device).double().cpu()
    want, tolerance = expected(b)
    cu = b["cu_seqlens_q"].tolist()
    for s, (held, new) in enumerate(MIXED):
        if held <= 40:
            rows = slice(cu[s], cu[s + 1])
            assert ((out[rows] - want[rows]).abs() <= tolerance[rows]).all()


def test_two_calls_give_the_same_bits(device):
    b = on(rolling_batch(DECODES + CHUNKS, 200, 4, dtype=torch.bfloat16, kv_dtype=torch.float8_e4m3fn), device)
    first = call(b, device).clone()
    for _ in range(5):
        assert torch.equal(call(b, device), first)
