"""Oracle for a step of beam search, in fp64 and Python's order.

Test infrastructure only: see oracle/__init__.py.
"""
from __future__ import annotations

import math

import torch


def select(logits, scores, count):
    """(scores fp64, beams, tokens) [B, count] of logits [B W, V], scores [B, W].
    NaN first, then by score; the lowest (beam, token) among equals."""
    B, W = scores.shape
    V = logits.shape[1]
    out = ([], [], [])
    for b in range(B):
        x = logits[b * W:(b + 1) * W].double()
        lp = torch.log_softmax(x, -1)
        lp[torch.isneginf(x).all(-1)] = -math.inf  # a row of -inf alone
        s = scores[b].double()[:, None] + lp
        s[scores[b] == -math.inf] = torch.where(lp[scores[b] == -math.inf].isnan(), lp[scores[b] == -math.inf], -math.inf)
        flat = s.flatten()
        order = torch.sort(torch.where(flat.isnan(), math.inf, flat), descending=True, stable=True).indices[:count]
        out[0].append(flat[order])
        out[1].append(order // V)
        out[2].append(order % V)
    return tuple(torch.stack(o) if o else torch.zeros(0, count) for o in out)


def score_bound(logits, scores, want):
    """Largest error of a score: e^x in fp32 is off by a factor within 1 +- (2 + |x|) u,
    u = 2^-24 (the scaling by log2 e of an argument |x| rounds), which sum |x| e^x /
    sum e^x <= ln V weighs by at most 1 + ln V; 32 terms of a thread and 8 joins add 40 u;
    the rest is fp64, and one rounding to fp32."""
    u = 2.0 ** -24
    V = logits.shape[-1]
    finite = torch.where(torch.isfinite(want), want.abs(), torch.zeros_like(want))
    return (44 + 2 * math.log(V)) * u + u * finite * 1.01
