"""The paged model with a sliding window and sinks, through the engine: greedy tokens against the
float64 recompute under the window's mask, with the PyTorch path and with the kernels."""

from __future__ import annotations

import pytest
import torch

from engine_helpers import assert_tokens_match, make_engine, prompts, tiny_config
from mini_vllm.kernels import ops
from mini_vllm.model import random_weights
from mini_vllm.serve import SchedulerConfig
from oracle.qwen3_dense import generate_greedy

WINDOWS = [(1, 0), (16, 3), (7, 20), (500, 0)]
NEW = 12


def config_of(window, sinks, **over):
    return tiny_config(sliding_window=window, attention_sinks=sinks, **over)


def requests():
    return prompts(5, 3, 60, 512, seed=4)


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("chunk", [8, 512])
def test_engine_matches_the_windowed_recompute(window, sinks, chunk):
    config = config_of(window, sinks)
    weights = random_weights(config, seed=3, std=0.1)
    engine = make_engine(config, weights, sched=SchedulerConfig(max_batched_tokens=64, chunk_size=chunk))
    got = engine.generate(requests(), NEW)
    for prompt, tokens in zip(requests(), got):
        want, logits = generate_greedy(config, weights, prompt, NEW)
        tie = 1e-4 * max(1.0, float(torch.stack(logits).abs().max()))
        assert_tokens_match(tokens, want, logits, tie, f"window {window} sinks {sinks}")


def test_a_window_changes_the_tokens():
    config = config_of(4, 0)
    weights = random_weights(config, seed=3, std=0.1)
    prompt = requests()[0]
    assert len(prompt) > 8
    narrow = generate_greedy(config, weights, prompt, NEW)[0]
    assert narrow != generate_greedy(tiny_config(), weights, prompt, NEW)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("graphs", [False, True])
def test_kernels_match_the_windowed_recompute(extension, device, window, sinks, head_dim, graphs):
    config = config_of(window, sinks, head_dim=head_dim)
    weights = random_weights(config, seed=3, std=0.1)
    on_gpu = {k: v.to(device) for k, v in weights.items()}
    engine = make_engine(config, on_gpu, use_cuda=True, device=device, use_graphs=graphs)
    got = engine.generate(requests(), NEW)
    for prompt, tokens in zip(requests(), got):
        want, logits = generate_greedy(config, weights, prompt, NEW)
        tie = 1e-4 * max(1.0, float(torch.stack(logits).abs().max()))
        assert_tokens_match(tokens, want, logits, tie, f"window {window} sinks {sinks}")


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_kernels_match_the_torch_path_in_bf16(extension, device, kv_dtype):
    """Logits of whole prompts and of a chunk and one token after them, kernels on and off."""
    from mini_vllm.serve.batch import ForwardBatch
    from mini_vllm.serve.sequence import Sequence

    config = config_of(20, 5, head_dim=128, dtype=torch.bfloat16)
    weights = {k: v.to(device) for k, v in random_weights(config, seed=3, std=0.1).items()}
    logits = []
    for use_cuda in (True, False):
        engine = make_engine(config, weights, use_cuda=use_cuda, device=device, kv_dtype=kv_dtype)
        with ops.strict_kernels(use_cuda):
            seqs = [Sequence(i, tokens + [1, 2, 3, 4], 4) for i, tokens in enumerate(requests()[:2])]
            rows = []
            for new in (lambda s: len(s.prompt) - 4, lambda s: 3, lambda s: 1):
                step = [(s, new(s)) for s in seqs]
                for s, n in step:
                    engine.model.manager.allocate(s.seq_id, s.num_computed_tokens + n)
                rows.append(engine.model(ForwardBatch.from_scheduled(step, engine.model.manager, device)))
                for s, n in step:
                    s.num_computed_tokens += n
            logits.append(torch.cat(rows).float())
    # eight roundings of half a step a layer and stream, bfloat16, relative to the logits' size
    assert (logits[0] - logits[1]).abs().max() <= 16 * 2.0**-8 * logits[1].abs().max()
