"""The best continuations of a step of beam search.  The reference has no beam
search."""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from .. import _lib
from .fused_ops import compiler_disable

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
def _call(name, count, logits, scores):
    """The checks of a call of these layouts (_lib.layout), once: what it is launched with
    beside addresses, and the bytes of scratch.  On the tensors' device, which is current."""
    (_, dtype, shape, strides), (_, score_dtype, score_shape, _) = logits, scores
    if len(shape) != 2 or len(score_shape) != 2 or score_shape.numel() != shape[0]:
        raise ValueError(f"{name}: logits must be [texts * W, V] and scores [texts, W], got {tuple(shape)} and "
                         f"{tuple(score_shape)}")
    if score_dtype != torch.float32:
        raise ValueError(f"{name}: scores must be float32, got {score_dtype}")
    (B, W), V = score_shape, shape[1]
    if W == 0 or W > MAX_BEAMS or not 1 <= count <= min(MAX_COUNT, W * V):
        raise ValueError(f"{name}: {count} of {W} beams' continuations by {V} tokens (at most {MAX_COUNT} of "
                         f"{MAX_BEAMS} beams')")
    if dtype not in _lib._DTYPE_CODE:
        raise TypeError(f"hydra_amd: unsupported dtype {dtype}")
    code = _lib._DTYPE_CODE[dtype]
    need = ctypes.c_int64(0)
    _lib.call("hydra_beam_select_workspace", B, W, V, count, code, ctypes.byref(need))
    rows = (strides[1] == 1 or V == 1) and (strides[0] >= V or B * W <= 1)
    return rows, (strides[0] if rows and B * W > 1 else V), (B, W, V, count), code, need.value, _lib.load().hydra_beam_select


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
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError(f"{name}: no gradient (call it under torch.no_grad())")
    _lib.refuse_tangents(name, logits, scores)
    with _lib.on_device(logits):
        rows, stride, sizes, code, need, entry = _call(name, int(count), _lib.layout(logits), _lib.layout(scores))
        x, scores = logits if rows else logits.contiguous(), scores.contiguous()
        B, n = sizes[0], sizes[3]
        best = x.new_empty((B, n), dtype=torch.float32)
        beams, tokens = x.new_empty((2, B, n), dtype=torch.int64).unbind(0)
        parents = x.new_empty((B, n), dtype=torch.int32)
        ws = _lib.scratch(need, x)
        rc = entry(x.data_ptr(), stride, scores.data_ptr(), *sizes, best.data_ptr(), beams.data_ptr(), tokens.data_ptr(),
                   parents.data_ptr(), code, ws.data_ptr(), need, _lib.stream(x))
    _lib.check(rc, "hydra_beam_select")
    return BeamChoice(best, beams, tokens, parents)
