"""The best continuations of a step of beam search.  The reference has no beam
search."""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from .. import _lib
from .fused_ops import _as_rows, compiler_disable

MAX_BEAMS, MAX_COUNT = 1024, 128


class BeamChoice(NamedTuple):
    """Best first, [texts, count]: fp32 `scores`; int64 `beams` (within the text)
    and `tokens`; int32 `rows`, the logits' rows that they go on from (what
    PagePool.fork and take_rows take, as one vector)."""
    scores: torch.Tensor
    beams: torch.Tensor
    tokens: torch.Tensor
    rows: torch.Tensor


@functools.lru_cache(maxsize=1024)
def _workspace(device: int, *sizes) -> int:
    """Scratch bytes of these sizes on a device, which is current."""
    need = ctypes.c_int64(0)
    _lib.call("hydra_beam_select_workspace", *sizes, ctypes.byref(need))
    return need.value


@compiler_disable
def beam_select(logits: torch.Tensor, scores: torch.Tensor, count: int) -> BeamChoice:
    """The `count` (at most 128) best of each text's continuations, by
    scores[b, w] + ln softmax(logits[b W + w])[v] over its W beams (at most 1024)
    and the V tokens.

    logits [texts * W, V] (bf16, fp16 or fp32; rows at one stride from each other,
    others are copied first), scores fp32 [texts, W].  Among equals the lowest beam,
    then the lowest token comes first; scores are compared in fp64, from fp32 sums of
    exponentials.  Masked logits may be -inf or the type's lowest value, and the score of
    a beam that does not count yet -inf.  NaN counts as larger than any number; a row
    with a NaN or +inf has NaN throughout.  Inference only: no gradient."""
    name = "beam_select"
    _lib.require_gpu(name, logits, scores)
    if logits.dim() != 2 or scores.dim() != 2 or scores.numel() != logits.shape[0]:
        raise ValueError(f"{name}: logits must be [texts * W, V] and scores [texts, W], got {tuple(logits.shape)} and "
                         f"{tuple(scores.shape)}")
    if scores.dtype != torch.float32:
        raise ValueError(f"{name}: scores must be float32, got {scores.dtype}")
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError(f"{name}: no gradient (call it under torch.no_grad())")
    _lib.refuse_tangents(name, logits, scores)
    (B, W), V, count = scores.shape, logits.shape[1], int(count)
    if W == 0 or W > MAX_BEAMS or not 1 <= count <= min(MAX_COUNT, W * V):
        raise ValueError(f"{name}: {count} of {W} beams' continuations by {V} tokens (at most {MAX_COUNT} of "
                         f"{MAX_BEAMS} beams')")
    code = _lib.dtype_code(logits)
    x, (rows, stride) = _as_rows(logits)
    if stride < V and rows > 1:  # rows that overlap: broadcast ones
        x, (rows, stride) = _as_rows(logits.contiguous())
    scores = scores.contiguous()
    best = x.new_empty((B, count), dtype=torch.float32)
    beams, tokens = x.new_empty((2, B, count), dtype=torch.int64).unbind(0)
    parents = x.new_empty((B, count), dtype=torch.int32)
    with _lib.on_device(x):
        need = _workspace(x.device.index, B, W, V, count, code)
        ws = _lib.scratch(need, x)
        _lib.call("hydra_beam_select", x.data_ptr(), stride, scores.data_ptr(), B, W, V, count, best.data_ptr(),
                  beams.data_ptr(), tokens.data_ptr(), parents.data_ptr(), code, _lib.ptr(ws), need, _lib.stream(x))
    return BeamChoice(best, beams, tokens, parents)
