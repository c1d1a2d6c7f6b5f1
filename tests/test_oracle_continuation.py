"""What keeps the oracle of shared prefixes, 8-bit pages and beams honest: exact
rationals, a bookkeeping model of the pages and sorted lists (CPU)."""
from __future__ import annotations

import math
import random
from fractions import Fraction

import pytest
import torch

from oracle import beam as ob
from oracle import paged as op


def _nearest_even(x: Fraction) -> int:
    low = math.floor(x)
    rest = x - low
    return low + (rest > Fraction(1, 2) or (rest == Fraction(1, 2) and low % 2 == 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantise_int8_is_the_rational_quotient_rounded(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 7, generator=g).mul(torch.exp(4 * torch.randn(40, 1, generator=g))).to(dtype)
    x[0] = 0
    x[1, 0], x[1, 1:] = 127.0, 63.5  # middles: to the even neighbour
    q, s = op.quantise(x, torch.int8)
    for row, got, scale in zip(x.tolist(), q.tolist(), s.tolist()):
        top = max(map(abs, row))
        # the quotient in fp64, then in fp32: twice rounded differs from once by no more than the last place
        assert abs(Fraction(scale) - Fraction(top) / 127) <= Fraction(top) / 127 * Fraction(1, 2 ** 24) * Fraction(101, 100) \
            or scale == 2.0 ** -126
        assert got == [_nearest_even(Fraction(v) / Fraction(scale)) for v in row]
        assert max(map(abs, got)) <= 127


def test_quantise_e4m3_is_torchs_rounding_under_the_least_scale():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(60, 9, generator=g).mul(torch.exp(5 * torch.randn(60, 1, generator=g)))
    x[0] = 0
    q, s = op.quantise(x, torch.float8_e4m3fn)
    top = x.abs().amax(-1)
    assert torch.equal(torch.frexp(s).mantissa, torch.full_like(s, 0.5))  # powers of two
    assert bool((top / s <= 448).all())
    assert bool(((2 * top / s > 448) | (s == 2.0 ** -126)).all())
    assert torch.equal((x / s[:, None]).to(torch.float8_e4m3fn).double(), q)


def test_quantise_of_rows_that_are_not_finite():
    x = torch.tensor([[1.0, math.inf], [math.nan, 2.0], [1.0, 2.0]])
    for kind in (torch.int8, torch.float8_e4m3fn):
        q, s = op.quantise(x, kind)
        assert torch.isnan(s).tolist() == [True, True, False] and not q[:2].any()
        assert torch.isnan(op.dequantise(q.to(kind), s)[:2]).all()


@pytest.mark.parametrize("seed", range(6))
def test_forks_keep_what_rows_hold(seed):
    """Random steps and forks: every row reads the tokens that it went on with, a page's
    holders are one more than `extra`, and no page is lost."""
    rng = random.Random(seed)
    N, P, page, pages = 6, 5, 16, 40
    lengths, table, stack, count, extra = [0] * N, [[-1] * P for _ in range(N)], list(range(pages)), pages, [0] * pages
    texts = [[] for _ in range(N)]
    memory = {}  # (page, row) -> token
    mark = 0
    for _ in range(60):
        new = [rng.choice([0, 1, 5, 17]) for _ in range(N)]
        slots, lengths, _, granted, count, table = op.plan(lengths, new, table, stack, count, page, 17)
        for i in range(N):
            for s in (s for s in slots[i] if s >= 0):
                mark += 1
                assert extra[s // page] == 0  # what is written has one holder
                memory[s // page, s % page] = mark
                texts[i].append(mark)
        parents = [rng.choice([-1, rng.randrange(N), rng.randrange(N), i]) for i in range(N)]
        lengths, table, stack, count, extra, sources, copies, taken, ok = op.fork(parents, lengths, table, stack, count, extra, page)
        before = dict(memory)
        for a, b in zip(sources, copies):
            assert (a < 0) == (b < 0)
            for r in range(page):
                if a >= 0 and (a, r) in before:
                    memory[b, r] = before[a, r]
        texts = [list(texts[t]) if t >= 0 else [] for t in taken]
        holders = [0] * pages
        for i in range(N):
            assert lengths[i] == len(texts[i])
            assert [memory[table[i][k // page], k % page] for k in range(lengths[i])] == texts[i]
            for p in table[i][:-(-lengths[i] // page)]:
                holders[p] += 1
        assert all(max(h - 1, 0) == e for h, e in zip(holders, extra))
        free = stack[:count]
        assert sorted(free + [p for p in range(pages) if holders[p]]) == list(range(pages))


def test_beam_selection_is_a_sorted_list():
    rng = random.Random(5)
    for B, W, V, n in ((1, 1, 5, 5), (2, 3, 7, 9), (3, 4, 2, 8)):
        logits = torch.tensor([[rng.choice([0.0, 1.0, -2.5, -math.inf]) for _ in range(V)] for _ in range(B * W)])
        logits[0] = -math.inf
        scores = torch.tensor([[rng.choice([0.0, -1.0, -math.inf]) for _ in range(W)] for _ in range(B)])
        s, beams, tokens = ob.select(logits, scores, n)
        for b in range(B):
            every = []
            for w in range(W):
                row = logits[b * W + w].tolist()
                total = sum(math.exp(x) for x in row)
                for v, x in enumerate(row):
                    score = float(scores[b, w]) + (x - math.log(total) if total > 0 and x > -math.inf else -math.inf)
                    every.append((-round(score, 9), w * V + v))
            every.sort()
            assert [(w * V + v) for w, v in zip(beams[b].tolist(), tokens[b].tolist())] == [i for _, i in every[:n]]
            assert all(a == b_ or abs(a + b_) < 1e-9 or a == -b_ for (a, _), b_ in zip(every, s[b].tolist()))
