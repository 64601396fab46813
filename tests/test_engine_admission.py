"""Admissions of the dense engine whose prompts all end with their first token, while
others still wait."""

import pytest
import torch

from distrl_llm_amd.config import SamplingParams
from test_chunked_prefill import _engine, _model, _prompts


@pytest.mark.parametrize("session", [False, True])
def test_prompts_of_one_token_each(session, monkeypatch):
    if session:
        monkeypatch.setenv("DISTRL_FORCE_SESSION", "1")
    model = _model("tiny-qwen2", torch.device("cpu"), torch.float32)
    engine = _engine(model, 0, cache=True)
    prompts = _prompts((9,) * 70, 2048)         # 32 fit at a time
    sp = SamplingParams(max_tokens=1, temperature=0.0, n=1)
    got = engine.generate(prompts, sp, eos_token_id=None)
    assert got == [engine.generate([p], sp, eos_token_id=None)[0] for p in prompts]
    limits = [[1]] * 40 + [[3]] + [[1]] * 29
    got = engine.generate(prompts, SamplingParams(max_tokens=3, temperature=0.0, n=1),
                          eos_token_id=None, token_limits=limits)
    assert [len(c) for per in got for c in per] == [n for per in limits for n in per]
    engine.clear_prefix_cache()
    assert engine.pool.allocator.num_free == engine.pool.num_blocks


def test_a_pool_that_is_too_small():
    model = _model("tiny-qwen2", torch.device("cpu"), torch.float32)
    engine = _engine(model, 0)
    held = [engine.pool.allocator.alloc() for _ in range(engine.pool.num_blocks - 1)]
    with pytest.raises(MemoryError, match="pool"):
        engine.generate(_prompts((9, 40), 2048), SamplingParams(max_tokens=9, n=1),
                        eos_token_id=None)
    assert held
