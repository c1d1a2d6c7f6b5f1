"""What keeps the serving oracle honest: library identities, autograd and a
bookkeeping model of the pages (CPU)."""
from __future__ import annotations

import random

import pytest
import torch
import torch.nn.functional as F

from oracle import logprobs as ol
from oracle import paged as op

INF = float("inf")


@pytest.mark.parametrize("seed", range(4))
def test_pages_are_held_once_and_come_back(seed):
    """Random steps: no page is held twice or lost, tokens keep their slots."""
    rng = random.Random(seed)
    N, P, page, pages = 5, 6, 16, 14
    lengths, table, stack, count = [0] * N, [[-1] * P for _ in range(N)], list(range(pages)), pages
    held = [[] for _ in range(N)]  # the slot of each token
    for _ in range(40):
        new = [rng.choice([0, 1, 1, 7, 30]) for _ in range(N)]
        slots, after, seen, granted, count, table = op.plan(lengths, new, table, stack, count, page, 30)
        room = count
        for i in range(N):
            got = [s for s in slots[i] if s >= 0]
            assert len(got) == (new[i] if granted[i] else 0) and after[i] == lengths[i] + len(got)
            assert seen[i] == (after[i] if got else 0)
            held[i] += got
            need = -(-(lengths[i] + new[i]) // page) - -(-lengths[i] // page)
            assert granted[i] or lengths[i] + new[i] > P * page or need > room - sum(not g for g in granted[:i])
        lengths = after
        done = [rng.random() < 0.2 for _ in range(N)]
        lengths, table, stack, count = op.release(done, lengths, table, stack, count, page)
        held = [[] if d else h for h, d in zip(held, done)]
        flat = [s for h in held for s in h]
        assert len(set(flat)) == len(flat)
        used = [table[i][c] for i in range(N) for c in range(-(-lengths[i] // page))]
        assert sorted(used + stack[:count]) == list(range(pages))
        for i, h in enumerate(held):
            assert h == [table[i][t // page] * page + t % page for t in range(lengths[i])]


def test_a_request_that_finds_no_room_holds_back_those_behind_it():
    slots, after, _, granted, count, _ = op.plan([0, 0, 3], [40, 5, 1], [[-1] * 4] * 2 + [[4, -1, -1, -1]], [0, 1], 2, 16, 40)
    assert granted == [False, False, True] and after == [0, 0, 4] and count == 2 and slots[2][0] == 4 * 16 + 3


@pytest.mark.parametrize("H,K", [(4, 4), (6, 2)])
def test_attention_is_softmax_over_the_gathered_rows(H, K):
    g = torch.Generator().manual_seed(H)
    q, kp, vp = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, H, 8), (5, K, 16, 8), (5, K, 16, 8)))
    table = torch.tensor([[3, 0, 4], [1, 9, 2]], dtype=torch.int32)  # 9: outside the pool
    out, weight = op.attention(q, kp, vp, table, torch.tensor([37, 48]), scale=0.3)
    for n, ids, drop in ((0, [3, 0, 4], slice(37, 48)), (1, [1, 2], slice(0, 0))):
        k, v = (torch.cat([t[i] for i in ids], 1) for t in (kp, vp))
        mask = torch.zeros(k.shape[1], dtype=torch.float64)
        mask[drop] = -INF
        k, v = (t.repeat_interleave(H // K, 0) for t in (k, v))
        want = F.scaled_dot_product_attention(q[n][:, None], k, v, attn_mask=mask[None], scale=0.3)[:, 0]
        assert torch.allclose(out[n], want, rtol=1e-12, atol=1e-13)
    assert bool((weight >= out.abs() - 1e-12).all())
    assert not op.attention(q, kp, vp, table, torch.tensor([0, -3]))[0].any()


@pytest.mark.parametrize("T", [1.0, 0.7])
def test_logprobs_and_their_gradient(T):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 40, generator=g, dtype=torch.float64) * 2
    x[2, 5:30] = -INF
    tokens = torch.tensor([3, 0, 4, -100, 39, 40])
    logp, entropy, top, ids = ol.forward(x, tokens, 4, T)
    dist = torch.distributions.Categorical(logits=(x[[0, 1, 3, 4, 5]] / T))
    assert torch.allclose(entropy[[0, 1, 3, 4, 5]], dist.entropy(), rtol=1e-12)
    want = torch.log_softmax(x / T, 1)
    assert torch.allclose(logp[[0, 1, 2, 4]], want[[0, 1, 2, 4], [3, 0, 4, 39]], rtol=1e-12) and not logp[[3, 5]].any()
    assert torch.equal(top, want.topk(4).values) and torch.equal(ids, want.topk(4).indices)

    gl, gh, gt = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6,), (6,), (6, 4)))
    leaf = x.clone().requires_grad_()
    lp = torch.log_softmax(leaf / T, 1)
    shown = torch.where(lp == -INF, torch.zeros_like(lp), lp)
    taken = lp.gather(1, tokens.clamp(0, 39)[:, None])[:, 0] * ((tokens >= 0) & (tokens < 40))
    ((taken * gl).sum() - ((lp.exp() * shown).sum(1) * gh).sum() + (lp.gather(1, ids) * gt).sum()).backward()
    got = ol.backward(x, tokens, gl, gh, gt, ids, T)
    keep = x != -INF
    assert torch.allclose(got[keep], leaf.grad[keep], rtol=1e-10, atol=1e-12) and not got[~keep].any()


def test_logprobs_of_rows_without_a_logit_and_equal_ones():
    x = torch.full((2, 7), -INF)
    x[1] = 2.5
    logp, entropy, top, ids = ol.forward(x, torch.tensor([1, 6]), 3)
    assert logp[0] == -INF and entropy[0] == 0 and ids.tolist() == [[0, 1, 2]] * 2
    assert torch.allclose(entropy[1], torch.tensor(7.0).double().log()) and torch.allclose(logp[1], -entropy[1])
    grad = ol.backward(x, torch.tensor([1, 6]), torch.ones(2), torch.ones(2))
    # seven terms below 1, each of a logarithm, an exponential and four products and
    # sums in fp64 (8 steps of 2^-53), and the six additions of their sum
    assert not grad[0].any() and abs(float(grad[1].sum())) <= (7 * 8 + 6) * 2.0 ** -53
