"""Oracle for log probabilities of tokens, entropy and top alternatives with
their gradient: fp64 from the definitions, and the bounds of an fp32
evaluation.

Test infrastructure only: see oracle/__init__.py.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def forward(logits, tokens, top_k=0, temperature=1.0):
    """(logprobs, entropy, top_logprobs, top_tokens) of logits [rows, V]."""
    z = logits.double() / temperature
    rows, V = z.shape
    logp = torch.zeros(rows, dtype=torch.float64)
    entropy = torch.zeros(rows, dtype=torch.float64)
    top = torch.full((rows, top_k), -float("inf"), dtype=torch.float64)
    ids = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top_k]
    for r in range(rows):
        given = 0 <= int(tokens[r]) < V
        if bool((z[r] == -float("inf")).all()):
            logp[r] = -float("inf") if given else 0.0
            continue
        lp = torch.log_softmax(z[r], 0)
        if given:
            logp[r] = lp[int(tokens[r])]
        entropy[r] = -torch.where(lp == -float("inf"), 0.0, lp.exp() * lp).sum()
        top[r] = lp[ids[r]]
    return logp, entropy, top, ids


def backward(logits, tokens, g_logp, g_entropy, g_top=None, top_tokens=None, temperature=1.0):
    """The gradient from the formula, [rows, V] fp64."""
    z = logits.double() / temperature
    rows, V = z.shape
    grad = torch.zeros(rows, V, dtype=torch.float64)
    for r in range(rows):
        if bool((z[r] == -float("inf")).all()):
            continue
        lp = torch.log_softmax(z[r], 0)
        p = lp.exp()
        plp = torch.where(p == 0, 0.0, p * lp)
        H = -plp.sum()
        t = int(tokens[r])
        gl = float(g_logp[r]) if 0 <= t < V else 0.0
        g = -(gl + (0.0 if g_top is None else float(g_top[r].double().sum()))) * p
        g -= float(g_entropy[r]) * (plp + p * H)
        if 0 <= t < V:
            g[t] += gl
        if g_top is not None:
            g[top_tokens[r]] += g_top[r].double()
        grad[r] = g / temperature
    return grad


def bounds(logits, tokens, top_tokens, temperature, g_logp=None, g_entropy=None, g_top=None):
    """Largest errors of (logprobs, entropy, top_logprobs, gradient) computed in
    fp32, of rows whose logits are finite or -inf.

    t = (x - M) log2(e) / T is off by 3 u of itself (difference, constant,
    product), so 2^t by a factor within 1 +- (3 |t| ln 2 + 2) u; a thread adds at
    most V / 512 + 8 of them and 9 partial sums follow: s is off by a factor
    within 1 +- ds, ds = (3 ln 2 E|t| + V / 512 + 20) u, E over the softmax.
    log2 is good to 2 u of itself (and u in s's neighbourhood of 1)."""
    V = logits.shape[1]
    x = logits.double()
    m = x.amax(1, keepdim=True)
    t = torch.where(x == -float("inf"), 0.0, (x - m) / temperature)  # ln units
    p = torch.softmax(x / temperature, 1)
    ls = torch.logsumexp((x - m) / temperature, 1)
    n = V / 512 + 20
    mean_t = (p * t.abs()).sum(1)
    ds = (3 * mean_t + n) * U
    dls = ds + 3 * U * ls.abs() + U
    dlp = lambda tt: 4 * U * tt.abs() + dls.view(-1, *[1] * (tt.dim() - 1)) + 4 * U * (tt.abs() + ls.abs().view(-1, *[1] * (tt.dim() - 1)))  # noqa: E731
    at = tokens.clamp(0, V - 1)[:, None]
    lp_bound = dlp(t.gather(1, at)[:, 0])
    dw = (p * t.abs() * (3 * t.abs() + 5)).sum(1) * U + (n * U + ds + 3 * U) * mean_t
    h_bound = dls + dw + 3 * U * (ls.abs() + mean_t)
    top_bound = dlp(t.gather(1, top_tokens))
    if g_logp is None:
        return lp_bound, h_bound, top_bound
    lp = t - ls[:, None]
    H = -(p * torch.where(p == 0, 0.0, lp)).sum(1, keepdim=True)
    given = ((tokens >= 0) & (tokens < V))[:, None]
    gl = torch.where(given, g_logp.double()[:, None].abs(), 0.0)
    gh = g_entropy.double()[:, None].abs()
    gt = torch.zeros_like(gl) if g_top is None else g_top.double().abs().sum(1, keepdim=True)
    size = gl + gt + gh * (t.abs() + 2 * ls.abs()[:, None] + H.abs())  # of A + B t and its terms
    inner = size * ((3 * t.abs() + 12 + top_tokens.shape[1]) * U + ds[:, None]) + gh * (h_bound + dls)[:, None]
    g_bound = p * inner / temperature
    g_bound.scatter_add_(1, at, torch.where(given, 4 * U * gl / temperature, 0.0))
    if g_top is not None:
        g_bound.scatter_add_(1, top_tokens, 4 * U * g_top.double().abs() / temperature)
        g_bound.scatter_add_(1, at, torch.where(given, 4 * U * gt / temperature, 0.0))
    return lp_bound, h_bound, top_bound, g_bound


__all__ = ["forward", "backward", "bounds"]
