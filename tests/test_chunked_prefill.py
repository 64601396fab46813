"""Prompt phases over a cache that holds tokens already: prefixes of earlier prompts,
chunks of the same prompt (EngineConfig.prefill_chunk_tokens)."""

import pytest
import torch

from distrl_llm_amd.config import EngineConfig, SamplingParams
from distrl_llm_amd.engine import Engine
from distrl_llm_amd.engine.kvcache import Sequence
from distrl_llm_amd.models import CausalLM, get_spec

LENGTHS = [(1,), (9, 40), (3, 64, 29, 1), (70, 8, 16)]


def _prompts(lengths, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def _model(name, device, dtype, lora_r=4):
    model = CausalLM(get_spec(name), lora_r=lora_r, lora_alpha=8, dtype=dtype,
                     device=device).random_init(11).eval()
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("lora_B"):
                p.copy_(torch.randn(p.shape, generator=g) * 0.05)
    return model


def _engine(model, chunk, cache=False, block=8, device="cpu"):
    return Engine(model, EngineConfig(
        max_seq_length=256, kv_block_size=block, num_kv_blocks=128, max_num_seqs=32,
        enable_prefix_caching=cache, prefill_chunk_tokens=chunk),
        device=torch.device(device), seed=0)


def _prefill(engine, prompts):
    if engine.fused is not None:
        engine.fused.refresh()
    seqs = [Sequence(i, p, i) for i, p in enumerate(prompts)]
    with torch.no_grad():
        logits = engine._prefill_batch(seqs)
    rows = [engine.pool.key[:, q.block_table].flatten(1, 2)[:, :q.context_len] for q in seqs]
    return logits, torch.cat(rows, 1)


@pytest.fixture(scope="module")
def tiny():
    return _model("tiny-qwen2", torch.device("cpu"), torch.float32)


@pytest.mark.parametrize("chunk", [1, 7, 8, 64])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_chunks_match_one_pass(tiny, lengths, chunk):
    """Logits and cached keys, two orders of the same fp32 sums of some hundred terms."""
    prompts = _prompts(lengths, 2048)
    want, got = (_prefill(_engine(tiny, c), prompts) for c in (0, chunk))
    for x, y in zip(got, want):
        assert float((x - y).abs().max()) <= 2.0 ** -14 * float(y.abs().max())


@pytest.mark.parametrize("chunk", [0, 5])
def test_cached_prefix_and_chunks_generate_alike(tiny, chunk):
    head = list(range(300, 333))
    prompts = [head + p for p in _prompts((1, 40, 7), 2048, 3)] + _prompts((11,), 2048, 4)
    sp = SamplingParams(max_tokens=5, temperature=0.0, n=2)
    want = _engine(tiny, 0).generate(prompts, sp, eos_token_id=None)
    engine = _engine(tiny, chunk, cache=True)
    engine.generate([head + [1, 2]], sp, eos_token_id=None)
    assert engine.generate(prompts, sp, eos_token_id=None) == want
    assert engine._prefix_hits >= 3 * 4
    engine.clear_prefix_cache()
    assert engine.pool.allocator.num_free == engine.pool.num_blocks


def test_steps_carry_the_budget(tiny, monkeypatch):
    engine, steps = _engine(tiny, 16), []
    step = engine._prefill_step
    monkeypatch.setattr(engine, "_prefill_step",
                        lambda seqs, new: steps.append(list(new)) or step(seqs, new))
    _prefill(engine, _prompts((20, 3, 30), 2048))
    assert steps == [[16], [4, 3, 9], [16], [5]]


def test_a_tail_runs_in_one_step(tiny, monkeypatch):
    engine = _engine(tiny, 0, cache=True)
    head = list(range(50, 90))
    _prefill(engine, [head])
    steps = []
    step = engine._prefill_step
    monkeypatch.setattr(engine, "_prefill_step",
                        lambda seqs, new: steps.append(list(new)) or step(seqs, new))
    _prefill(engine, [head + [1, 2, 3], [5, 6]])
    assert steps == [[3, 2]]


def test_refusals(tiny):
    with pytest.raises(ValueError, match="prefill_chunk_tokens"):
        _engine(tiny, -1)
    with pytest.raises(ValueError, match="token"):
        _engine(tiny, 0)._prefill_step([Sequence(0, [], 0)], [0])


@pytest.mark.gpu
@pytest.mark.parametrize("packs", [True, False])
@pytest.mark.parametrize("name,lora_r", [("small-qwen2", 0), ("small-qwen2", 32), ("small-qwen3", 8)])
def test_chunks_match_one_pass_gpu(name, lora_r, packs):
    """Two orders of the same products in bf16, as between the packed and the module
    path: 2 % of the norm."""
    model = _model(name, torch.device("cuda"), torch.bfloat16, lora_r)
    prompts = _prompts((150, 1, 64, 33), 4096)
    got = []
    for chunk in (0, 40, 64):
        engine = _engine(model, chunk, block=16, device="cuda")
        if not packs:
            engine._prefill_packs = lambda: False
        got.append(_prefill(engine, prompts))
    for other in got[1:]:
        for x, y in zip(other, got[0]):
            assert float((x - y).float().norm() / y.float().norm()) < 0.02


@pytest.mark.gpu
def test_cached_prefix_gpu():
    model = _model("small-qwen2", torch.device("cuda"), torch.bfloat16, 8)
    head = list(range(700, 800))
    prompts = [head + p for p in _prompts((1, 40, 7, 130), 4096, 3)] + _prompts((11,), 4096, 4)
    want, _ = _prefill(_engine(model, 0, block=16, device="cuda"), prompts)
    engine = _engine(model, 0, cache=True, block=16, device="cuda")
    _prefill(engine, [head])
    got, _ = _prefill(engine, prompts)
    assert engine._prefix_hits == 4 * 6
    assert float((got - want).float().norm() / want.float().norm()) < 0.02
