"""Bits of the softmax weights in the attention of chunks over a paged cache: what they lose
stays far below a bf16 step, as in the attention of single tokens.

Queries and keys are small whole numbers, so that scores are exact but for the scale: each
is off by 2^-22 of its size, which is below 16, and exp2 by a unit in the last place, so that
a weight in 32 bits is off by less than 2^-17 of itself. Two bf16 terms of it are off by
2^-16 at most. Sums of n weights and of n weighted values in 32 bits, whatever their order,
are off by n 2^-24 each at most. With the result's own rounding
|o - exact| <= 2^-8 |exact| + (2^-14 + n 2^-23) sum w |v|. Weights of one bf16 term are off by
up to 2^-8 each, and are beyond it at all of these sizes."""

import pytest
import torch

from distrl_llm_amd.ops import functional as OF
from test_chunk_ops import exact_fast, make

CASES = [
    dict(heads=14, kv=2, dim=64, new=[5], cached=[200]),            # few rows
    dict(heads=8, kv=2, dim=128, new=[2], cached=[300]),
    dict(heads=14, kv=2, dim=64, new=[5], cached=[1040]),           # in slices
    dict(heads=28, kv=4, dim=128, new=[1, 3], cached=[2000, 900]),
    dict(heads=14, kv=2, dim=64, new=[130, 17], cached=[40, 300]),  # more rows
    dict(heads=28, kv=4, dim=128, new=[40, 3], cached=[100, 9]),
    dict(heads=64, kv=8, dim=128, new=[640], cached=[1700]),        # many, a long context
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", CASES)
def test_weights_keep_their_bits(sizes):
    case = make(block=16, device="cuda", **sizes)
    g = torch.Generator().manual_seed(7)

    def whole(like):
        return torch.randint(-2, 3, like.shape, generator=g).to(like)

    key, value = case["key_cache"], case["value_cache"]
    case["q"] = whole(case["q"])
    case["key_cache"] = torch.where(key.isnan(), key, whole(key))
    case["value_cache"] = torch.where(value.isnan(), value, whole(value).sign())
    want, size = exact_fast(**case)
    n = int(case["context_lens"].max())
    off = (OF.paged_attention_chunk(**case).cpu().double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + size * (2.0 ** -14 + n * 2.0 ** -23) + 1e-30
    assert bool((off <= bound).all()), float((off / bound).max())
