"""Lengths of any size in the layout of a step's cache rows: sums of tokens and pages past
2^31 neither wrap nor run for ever, and what rows, tables and pages there are get theirs."""

import pytest
import torch

from distrl_llm_amd.ops import functional as OF

MOST = 2 ** 31 - 1

CASES = [
    dict(ctx=[0], new=[MOST], block=1),
    dict(ctx=[0], new=[MOST - 200_000], block=1),
    dict(ctx=[0, 3, 0], new=[MOST, 7, MOST], block=1),
    dict(ctx=[0, 0, 0, 5], new=[2 ** 30, 2 ** 30, 3, 2], block=1),
    dict(ctx=[MOST - 1, 3, 5], new=[1, 2, 1], block=1, held=[0, 0, 9]),
    dict(ctx=[2, MOST - 9, 4], new=[9, 9, 9], block=16, held=[0, MOST, 0]),
    dict(ctx=[4] * 600, new=[MOST] * 600, block=16),
    dict(ctx=[4] * 600, new=[0] * 599 + [MOST], block=3),
]


def oracle(tables, ctx, new, pages, block, rows, held):
    """By arithmetic, row by row and table entry by table entry."""
    width, cu, opened = len(tables[0]), [0], [0]
    have = [-(-c // block) for c in ctx] if held is None else held
    need = [max(0, -(-(c + n) // block) - h) for c, n, h in zip(ctx, new, have)]
    for n, m in zip(new, need):
        cu.append(cu[-1] + n)
        opened.append(opened[-1] + m)

    def entry(b, p):
        at = opened[b] + p - have[b]
        if not have[b] <= p < have[b] + need[b]:
            return tables[b][p]
        return pages[at] if at < len(pages) else -1

    after = [[entry(b, p) for p in range(width)] for b in range(len(ctx))]
    positions, slots = [], []
    for i in range(rows):
        b = max((b for b in range(len(ctx)) if cu[b] <= i < cu[b + 1]), default=None)
        position = 0 if b is None else ctx[b] + i - cu[b]
        page = -1 if b is None or position // block >= width else after[b][position // block]
        positions.append(position)
        slots.append(page * block + position % block if page >= 0 else -1)
    return positions, slots, [min(c, rows) for c in cu], \
        [min(max(c, 1), rows) - 1 for c in cu[1:]], after


def check(device, ctx, new, block, held=None, rows=20, width=4):
    tables = [[100 * b + p + 7 for p in range(width)] for b in range(len(ctx))]
    pages = list(range(90_000, 90_000 + 3 * len(ctx)))
    want = oracle(tables, ctx, new, pages, block, rows, held)

    def t(x):
        return torch.tensor(x, dtype=torch.int32, device=device)

    got_tables = t(tables)
    got = OF.chunk_slots(got_tables, t(ctx), t(new), t(pages), block, rows,
                         None if held is None else t(held))
    for x, y in zip((got.positions, got.slots, got.cu, got.last, got_tables), want):
        assert x.tolist() == y


@pytest.mark.parametrize("case", CASES)
def test_lengths_cpu(case):
    check("cpu", **case)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_lengths(case):
    check("cuda", **case)
