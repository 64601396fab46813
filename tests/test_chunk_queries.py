"""Queries that are no finite numbers in the attention of chunks over a paged cache: the
row and head they are in is no number, whichever kernel takes it, and no other is touched."""

import math

import pytest
import torch

from distrl_llm_amd.ops import functional as OF
from test_chunk_ops import make

CASES = [
    dict(heads=14, kv=2, dim=64, new=[5, 3], cached=[200, 0]),      # few rows
    dict(heads=8, kv=2, dim=128, new=[4], cached=[100]),
    dict(heads=14, kv=2, dim=64, new=[5], cached=[1040]),           # in slices
    dict(heads=8, kv=2, dim=128, new=[4], cached=[5000]),
    dict(heads=28, kv=4, dim=128, new=[1, 3], cached=[2000, 900]),
    dict(heads=14, kv=2, dim=64, new=[130, 17], cached=[40, 300]),  # more rows
    dict(heads=28, kv=4, dim=128, new=[40, 3], cached=[100, 9]),
    dict(heads=64, kv=8, dim=128, new=[640], cached=[1700]),        # many, a long context
]


def check(case, value):
    want = OF.paged_attention_chunk(**case)
    rows, heads = case["q"].shape[:2]
    hit = torch.zeros(rows, heads, dtype=torch.bool, device=want.device)
    q = case["q"].clone()
    for row, head in ((0, 1), (rows // 2, 0), (rows - 1, heads - 1)):
        q[row, head, row % q.shape[2]] = value
        hit[row, head] = True
    got = OF.paged_attention_chunk(**{**case, "q": q})
    assert bool(got[hit].isnan().all())
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_that_are_no_numbers_cpu(value):
    check(make(4, 2, 16, 8, [5, 40, 1], [30, 0, 9], dtype=torch.float32), value)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("sizes", CASES)
def test_queries_that_are_no_numbers(sizes, value):
    check(make(block=16, device="cuda", **sizes), value)


@pytest.mark.gpu
def test_no_key_and_no_number():
    """A row that sees no key is zeros whatever its query, as are rows of no sequence."""
    for new, context in (([4, 5], [2, 3]), ([300], [100])):
        case = make(8, 2, 64, 16, new, [0] * len(new), device="cuda", pad_rows=3)
        case["context_lens"] = torch.tensor(context, dtype=torch.int32, device="cuda")
        case["q"] = torch.full_like(case["q"], math.nan)
        got = OF.paged_attention_chunk(**case)
        first = 0
        for n, c in zip(new, context):
            assert not bool(got[first:first + n - c].any())
            assert bool(got[first + n - c:first + n].isnan().all())
            first += n
        assert not bool(got[first:].any())
