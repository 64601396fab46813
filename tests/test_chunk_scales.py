"""The scales that the attention of chunks over a paged cache takes, and those it refuses.

Queries and keys are whole numbers up to 2, so scores are exact before they are scaled. With
a scale of 1e6 they differ by 0 or far more than a weight's range, so that a row is the mean
of the values at its best score; with 1e-12 all weights are alike to 2^-29. What is left of
the error is the result's rounding, 2^-8 of it at most, the weights' (two terms, 2^-16) and
that of sums of n terms in 32 bits, n 2^-23, all of the sum of w |v|."""

import math

import pytest
import torch

from distrl_llm_amd.ops import functional as OF
from test_chunk_ops import exact_fast, make

ENDS = [1e-12, 1e6]


def check(case):
    g = torch.Generator().manual_seed(3)

    def whole(like):
        return torch.randint(-2, 3, like.shape, generator=g).to(like)

    case["q"] = whole(case["q"])
    case["key_cache"] = torch.where(case["key_cache"].isnan(), math.nan,
                                    whole(case["key_cache"]))
    want, size = exact_fast(**case)
    n = int(case["context_lens"].max())
    off = (OF.paged_attention_chunk(**case).cpu().double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + size * (2.0 ** -15 + n * 2.0 ** -23) + 1e-30
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("scale", ENDS)
def test_ends_cpu(scale):
    check({**make(4, 2, 16, 8, [5, 40, 1], [30, 0, 9], dtype=torch.float32), "scale": scale})


@pytest.mark.gpu
@pytest.mark.parametrize("scale", ENDS)
@pytest.mark.parametrize("sizes", [
    dict(heads=14, kv=2, dim=64, new=[5, 3], cached=[200, 0]),      # few rows
    dict(heads=8, kv=2, dim=128, new=[4], cached=[5000]),           # in slices
    dict(heads=28, kv=4, dim=128, new=[40, 3], cached=[100, 9]),    # more rows
    dict(heads=64, kv=8, dim=128, new=[640], cached=[1700]),        # many, a long context
])
def test_ends(sizes, scale):
    check({**make(block=16, device="cuda", **sizes), "scale": scale})


def test_refusals_cpu():
    case = make(4, 2, 16, 4, [3], [2], dtype=torch.float32)
    for scale in (1e-30, 0.99e-12, 1.01e6, 1e29):
        with pytest.raises(ValueError, match="scale"):
            OF.paged_attention_chunk(**{**case, "scale": scale})


@pytest.mark.gpu
def test_refusals():
    from distrl_llm_amd.ops.build import get_extension
    case = make(8, 2, 64, 16, [4, 5], [20, 0], device="cuda")
    for scale in (1e-30, 0.99e-12, 1.01e6, 1e29, math.nan, -1.0):
        with pytest.raises(ValueError, match="scale"):
            OF.paged_attention_chunk(**{**case, "scale": scale})
        with pytest.raises(RuntimeError, match="scale"):
            get_extension().paged_attention_chunk(
                *(case[n] for n in ("q", "key_cache", "value_cache", "block_tables", "cu",
                                    "context_lens")), scale, 5)
