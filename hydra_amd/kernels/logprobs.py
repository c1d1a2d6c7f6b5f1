"""Log probabilities of given tokens with the entropy and the top alternatives
of their rows: what a server returns beside a sampled token, and, with its
gradient, what a policy is trained on.  The reference has the mean
cross-entropy alone (chunked_cross_entropy)."""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .fused_ops import _as_rows, compiler_disable

MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    """fp32 `logprobs` and `entropy` [...], `top_logprobs` [..., k] (fp32) and
    `top_tokens` [..., k] (int64)."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def _forward(logits, tokens, top_k, temperature, want_stats):
    """(logits as rows, their number and stride, tokens in rows, the four
    results, stats)."""
    x, (rows, stride) = _as_rows(logits)
    if x.dim() > 1 and stride < x.shape[-1] and rows > 1:  # rows that overlap: broadcast ones
        x, (rows, stride) = _as_rows(logits.contiguous())
    tokens = tokens.reshape(-1).contiguous()  # a reshaped view may keep its stride
    lead = logits.shape[:-1]
    logp, entropy = (x.new_empty(lead, dtype=torch.float32) for _ in range(2))
    top = x.new_empty((*lead, top_k), dtype=torch.float32)
    ids = x.new_empty((*lead, top_k), dtype=torch.int64)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if want_stats else None
    with _lib.on_device(x):
        _lib.call("hydra_token_logprobs", x.data_ptr(), rows, x.shape[-1], stride, tokens.data_ptr(), temperature,
                  top_k, logp.data_ptr(), entropy.data_ptr(), _lib.ptr(stats), top.data_ptr(), ids.data_ptr(),
                  _lib.dtype_code(x), _lib.stream(x))
    return x, rows, stride, tokens, (logp, entropy, top, ids), stats


class _TokenLogprobsFunction(torch.autograd.Function):
    """Forward hydra_token_logprobs, backward hydra_token_logprobs_bwd."""

    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature):
        ctx.set_materialize_grads(False)
        x, _, _, tokens, out, stats = _forward(logits, tokens, top_k, temperature, True)
        ctx.save_for_backward(x, tokens, stats, out[1], out[3])
        ctx.meta = (top_k, temperature)
        ctx.mark_non_differentiable(out[3])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        x, tokens, stats, entropy, ids = ctx.saved_tensors
        top_k, temperature = ctx.meta
        _lib.refuse_tangents("token_logprobs", g_logp, g_entropy, g_top)
        _, (rows, stride) = _as_rows(x)
        if g_top is not None and top_k == 0:
            g_top = None
        g_logp, g_entropy, g_top = (None if g is None else g.float().contiguous() for g in (g_logp, g_entropy, g_top))
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        with _lib.on_device(x):
            _lib.call("hydra_token_logprobs_bwd", x.data_ptr(), rows, x.shape[-1], stride, tokens.data_ptr(),
                      temperature, top_k, stats.data_ptr(), entropy.data_ptr(), _lib.ptr(ids), _lib.ptr(g_logp),
                      _lib.ptr(g_entropy), _lib.ptr(g_top), grad.data_ptr(), _lib.dtype_code(x), _lib.stream(x))
        return grad, None, None, None


@compiler_disable
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """ln softmax(logits / temperature) at `tokens`, its entropy, and its
    `top_k` (at most 64) largest entries.

    logits [..., V] (bf16, fp16 or fp32), tokens [...] int64.  Rows may start
    anywhere, at one stride from each other; others (a batch's logits[:, :-1])
    are copied first, and the copy is kept for the backward.  A token outside
    [0, V) (an ignored position's -100) has the log probability 0 and no
    gradient through it; its row's entropy and alternatives are given as ever.
    Among equal logits the lowest index comes first.  Masked logits may be -inf
    or the type's lowest value; a row of -inf alone has log probabilities -inf,
    entropy 0 and no gradient; a row with a NaN or +inf has NaN.  A row that has
    masked or equal logits among its alternatives, and more than 1024 of them,
    takes a scan for each alternative.  The gradient covers logprobs, entropy
    and top_logprobs (once differentiable; forward-mode tangents are refused); a
    captured backward belongs to a captured forward, through
    torch.autograd.grad or leaves that no eager graph shares."""
    name = "token_logprobs"
    _lib.require_gpu(name, logits, tokens)
    _lib.refuse_tangents(name, logits)
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{name}: tokens {tuple(tokens.shape)} do not match logits {tuple(logits.shape)}")
    if tokens.dtype != torch.int64:
        raise ValueError(f"{name}: tokens must be int64, got {tokens.dtype}")
    V, top_k, temperature = logits.shape[-1], int(top_k), float(temperature)
    if not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"{name}: top_k must be in [0, min({MAX_TOP_K}, {V})], got {top_k}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"{name}: temperature must be positive and finite, got {temperature}")
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobsFunction.apply(logits, tokens, top_k, temperature))
    return TokenLogprobs(*_forward(logits, tokens, top_k, temperature, False)[4])
