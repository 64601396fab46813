"""What a prompt phase of the dense engine runs through, prompt by prompt: none is
computed another way because of what is cached of the others."""

import pytest
import torch

from distrl_llm_amd.ops import functional as OF
from test_chunked_prefill import _engine, _model, _prefill, _prompts

HEAD = list(range(300, 333))        # four whole pages of 8


@pytest.fixture(scope="module")
def tiny():
    return _model("tiny-qwen2", torch.device("cpu"), torch.float32)


def _with_head_cached(model, **kw):
    engine = _engine(model, 0, cache=True, **kw)
    _prefill(engine, [HEAD])
    return engine


MIXES = [(0, 1), (1, 0), (1, 0, 0, 1, 1), (0, 0, 1, 0)]       # 1: behind the cached head


def _mix(kinds):
    return [HEAD * kind + p
            for kind, p in zip(kinds, _prompts((9, 14, 3, 21, 6), 2048, len(kinds)))]


@pytest.mark.parametrize("kinds", MIXES)
def test_fresh_prompts_keep_their_attention(tiny, monkeypatch, kinds):
    """Beside cached ones they attend over their own rows, and logits come in the
    order of the prompts."""
    prompts = _mix(kinds)
    want, _ = _prefill(_engine(tiny, 0), prompts)
    engine = _with_head_cached(tiny)
    own, chunks = [], []
    attention, chunk = engine._prefill_attention, OF.paged_attention_chunk
    monkeypatch.setattr(engine, "_prefill_attention",
                        lambda q, k, v, lens: own.append(lens) or attention(q, k, v, lens))
    monkeypatch.setattr(OF, "paged_attention_chunk",
                        lambda q, *args: chunks.append(len(q)) or chunk(q, *args))
    got, _ = _prefill(engine, prompts)
    # two orders of the same fp32 sums of some hundred terms
    assert float((got - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max())
    layers = tiny.spec.num_layers
    assert own == [[len(p) for p, kind in zip(prompts, kinds) if not kind]] * layers
    assert chunks == [sum(len(p) - 32 for p, kind in zip(prompts, kinds) if kind)] * layers


@pytest.mark.gpu
@pytest.mark.parametrize("packs", [True, False])
@pytest.mark.parametrize("kinds", MIXES)
def test_fresh_prompts_beside_cached_ones_gpu(kinds, packs):
    """As between the packed and the module path: 2 % of the norm, row by row."""
    model = _model("small-qwen2", torch.device("cuda"), torch.bfloat16, 8)
    prompts = _mix(kinds)
    want, _ = _prefill(_engine(model, 0, device="cuda"), prompts)
    engine = _with_head_cached(model, device="cuda")
    if not packs:
        engine._prefill_packs = lambda: False
    got, _ = _prefill(engine, prompts)
    for x, y in zip(got.float(), want.float()):
        assert float((x - y).norm() / y.norm()) < 0.02


TAILS = [(1,), (2,), (1, 2, 1), (1,) * 20, (4,), (1, 2) * 6]


def _tails(lengths):
    return [HEAD[:32] + p for p in _prompts(lengths, 2048, 9)]


@pytest.mark.parametrize("lengths", TAILS)
def test_few_tokens_go_through_decode_steps(tiny, monkeypatch, lengths):
    """A token of each prompt a step, where that is the faster; more in one pass."""
    want, rows = _prefill(_engine(tiny, 0), _tails(lengths))
    engine, steps, passes = _with_head_cached(tiny), [], []
    step, chunk = engine._decode_forward, OF.paged_attention_chunk
    monkeypatch.setattr(engine, "_decode_forward",
                        lambda ids, *args: steps.append(len(ids)) or step(ids, *args))
    monkeypatch.setattr(OF, "paged_attention_chunk",
                        lambda q, *args: passes.append(len(q)) or chunk(q, *args))
    got, got_rows = _prefill(engine, _tails(lengths))
    by_steps = max(lengths) == 1 or max(lengths) == 2 and len(lengths) <= 8
    assert steps == ([sum(n > i for n in lengths) for i in range(max(lengths))]
                     if by_steps else [])
    assert passes == ([] if by_steps else [sum(lengths)] * tiny.spec.num_layers)
    for x, y in ((got, want), (got_rows, rows)):
        assert float((x - y).abs().max()) <= 2.0 ** -14 * float(y.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", TAILS)
def test_few_tokens_gpu(lengths):
    """As between decode and the prompt phase: 2 % of the norm, row by row."""
    model = _model("small-qwen2", torch.device("cuda"), torch.bfloat16, 8)
    want, _ = _prefill(_engine(model, 0, device="cuda"), _tails(lengths))
    got, _ = _prefill(_with_head_cached(model, device="cuda"), _tails(lengths))
    for x, y in zip(got.float(), want.float()):
        assert float((x - y).norm() / y.norm()) < 0.02


def test_sequences_end_where_they_are(tiny):
    """Tables, contexts and a generated token behind a tail of one."""
    from distrl_llm_amd.config import SamplingParams
    sp = SamplingParams(max_tokens=4, temperature=0.0, n=2)
    prompts = _tails((1, 1)) + [HEAD[:24] + [5]]
    want = _engine(tiny, 0).generate(prompts, sp, eos_token_id=None)
    engine = _with_head_cached(tiny)
    assert engine.generate(prompts, sp, eos_token_id=None) == want
    engine.clear_prefix_cache()


def test_only_prompts_that_end_have_logits(tiny, monkeypatch):
    """A chunk that does not end its prompt asks for no row of the vocabulary."""
    prompts = _prompts((20, 3, 30, 1), 2048)
    want, _ = _prefill(_engine(tiny, 0), prompts)
    engine, rows = _engine(tiny, 8), []
    logits = tiny.logits
    monkeypatch.setattr(tiny, "logits", lambda x: rows.append(len(x)) or logits(x))
    # steps of [8], [8], [4, 3, 1], [8], [8], [8], [5, 1]
    got, _ = _prefill(engine, prompts)
    assert rows == [2, 2]
    assert float((got - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max())
