"""A paged key-value cache: page tables planned on the GPU, key and value rows
stored into their pages and read back, the attention of one new token per
request over them, and requests that go on from what others hold.

A pool holds `k_pages` and `v_pages` [pages, Hkv, page_size, hd] (any strides
with a unit last one); position t of request i lies in page
`table[i, t // page_size]` at row `t % page_size`, and its *slot* is
`page * page_size + row`.  `page_size` is a power of two in [16, 4096].

Pages may be of 8 bits (torch.int8, torch.float8_e4m3fn), with a scale for
each row, fp32 [pages, Hkv, page_size]: a row stands for its values times it.

Nothing here synchronises with the host, so what only the device knows is
settled there: a request that finds no room is refused by the plan
(`granted`), a slot or table entry outside the pool stores and shows nothing.

The reference has no cache (it recomputes the sequence for every token).
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib


class PagePlan(NamedTuple):
    """What a step does with its requests: `slots` int64 [N, width] of the new
    tokens (-1 beside them), `positions` int32 [N] of the first ones,
    `lengths` int32 [N] afterwards, `seen` int32 [N] (the new length of the
    requests that got tokens, 0 of the others: what paged_attention takes),
    `granted` bool [N], `free_count` int32 [1] afterwards; `from_empty`: as
    the plan was asked for."""
    slots: torch.Tensor
    positions: torch.Tensor
    lengths: torch.Tensor
    seen: torch.Tensor
    granted: torch.Tensor
    free_count: torch.Tensor
    from_empty: bool = False


def _vector(name: str, what: str, t: torch.Tensor, dtype, n=None) -> torch.Tensor:
    if t.dtype != dtype or t.dim() != 1 or (n is not None and t.shape[0] != n):
        size = "" if n is None else f" of {n}"
        raise ValueError(f"{name}: {what} must be a {str(dtype)[6:]} vector{size}, got {t.dtype} {tuple(t.shape)}")
    return t


def _in_place(name: str, what: str, t: torch.Tensor, unit: bool = True) -> None:
    if unit and not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous (it is changed in place)")


def _check_table(name: str, table: torch.Tensor, n: int) -> None:
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != n:
        raise ValueError(f"{name}: table must be int32 [{n}, P], got {table.dtype} {tuple(table.shape)}")
    if (table.shape[1] > 1 and table.stride(1) != 1) or (n > 1 and table.stride(0) < table.shape[1]):
        raise ValueError(f"{name}: table needs rows of unit stride that do not overlap")


def _row_stride(table: torch.Tensor) -> int:
    """A lone row's stride says nothing."""
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def check_pages(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor) -> None:
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"{name}: k_pages and v_pages must be alike, [pages, Hkv, page_size, hd], got "
                         f"{tuple(k_pages.shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}")
    if 0 in k_pages.shape:
        raise ValueError(f"{name}: an empty pool {tuple(k_pages.shape)}")
    for t in (k_pages, v_pages):
        if not t.is_contiguous():
            check_distinct(name, "pages", t)


def check_no_gradient(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name}: no gradient (call it under torch.no_grad())")
    if _lib.forward_ad._current_level >= 0:
        _lib.refuse_tangents(name, *tensors)


def check_distinct(name: str, what: str, t: torch.Tensor) -> None:
    """A unit last stride, and no memory that two elements share."""
    reach = 1  # elements that the dimensions up to here span
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
        if size > 1 and stride < reach:
            raise ValueError(f"{name}: {what} of strides {t.stride()} overlap")
        reach += (size - 1) * stride
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: {what} need rows of unit stride")


def _strides(t: torch.Tensor):
    """Strides with a unit last one (torch gives a dimension of one element
    any)."""
    return _lib._stride_array((*t.stride()[:-1], 1)) if t.shape[-1] == 1 else _lib.strides(t)


def _plan(name, lengths, new_tokens, table, free_pages, free_count, page_size, width, from_empty,
          max_length=None, in_place=False):
    _lib.require_gpu(name, lengths, new_tokens, table, free_pages, free_count)
    N = _vector(name, "lengths", lengths, torch.int32).shape[0]
    _vector(name, "new_tokens", new_tokens, torch.int32, N)
    _vector(name, "free_pages", free_pages, torch.int32)
    _vector(name, "free_count", free_count, torch.int32, 1)
    _check_table(name, table, N)
    width = int(width)
    if N == 0 or table.shape[1] == 0 or width < 1:
        raise ValueError(f"{name}: {N} requests, {table.shape[1]} pages each, width {width}")
    lengths, new_tokens, free_pages = lengths.contiguous(), new_tokens.contiguous(), free_pages.contiguous()
    slots = lengths.new_empty((N, width), dtype=torch.int64)
    granted = lengths.new_empty((N,), dtype=torch.bool)
    after, seen, positions, left = lengths.new_empty((3 * N + 1,)).split((N, N, N, 1))
    if in_place:
        after, left = lengths, free_count
    within = () if max_length is None else (max_length,)
    with _lib.on_device(lengths):
        _lib.call("hydra_pool_plan" if within else "hydra_page_plan", lengths.data_ptr(), new_tokens.data_ptr(),
                  table.data_ptr(), _row_stride(table), free_pages.data_ptr(), free_pages.numel(),
                  free_count.data_ptr(), slots.data_ptr(), after.data_ptr(), seen.data_ptr(), granted.data_ptr(),
                  positions.data_ptr(), left.data_ptr(), N, table.shape[1], width, int(page_size), *within,
                  1 if from_empty else 0, _lib.stream(lengths))
    return PagePlan(slots, positions, after, seen, granted, left, bool(from_empty))


def plan_pages(lengths: torch.Tensor, new_tokens: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, width: int = 1, from_empty: bool = False) -> PagePlan:
    """Pages and slots of a step that adds `new_tokens[i]` (0 to `width`)
    tokens to request i, which holds `lengths[i]`.

    New pages come from the top of the stack `free_pages[:free_count]`, the
    requests served in order; their entries are written to `table` [N, P].
    A request is refused (its slots -1, its length unchanged) if it has more
    than `width` new tokens or no room for them in its table row, if the stack
    does not hold the pages that it and the requests before it need, or, with
    `from_empty`, if it adds to tokens that it holds already.  Lengths, new
    tokens and counts are int32 on the GPU, and stay as they are: copy
    `plan.lengths` and `plan.free_count` over them when the step is taken
    (PagePool does)."""
    return _plan("plan_pages", lengths, new_tokens, table, free_pages, free_count, page_size, width, from_empty)


def release_pages(done: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int, pages: Optional[int] = None) -> None:
    """Puts the pages of the requests with `done` (bool [N]) back on the
    stack, in place: their lengths become 0, their table entries -1.  Entries
    that are no page (negative, or not below `pages`, where that is given) do
    not come back.  A page belongs to one request: one that several tables name
    would come back more than once."""
    name = "release_pages"
    _lib.require_gpu(name, done, lengths, table, free_pages, free_count)
    N = _vector(name, "lengths", lengths, torch.int32).shape[0]
    _vector(name, "done", done, torch.bool, N)
    _vector(name, "free_pages", free_pages, torch.int32)
    _vector(name, "free_count", free_count, torch.int32, 1)
    _check_table(name, table, N)
    _in_place(name, "lengths", lengths)
    _in_place(name, "free_pages", free_pages)
    if N == 0 or table.shape[1] == 0 or free_pages.numel() == 0:
        return
    done = done.contiguous()
    within = () if pages is None else (int(pages),)
    with _lib.on_device(lengths):
        _lib.call("hydra_pool_release" if within else "hydra_page_release", done.data_ptr(), lengths.data_ptr(),
                  table.data_ptr(), _row_stride(table), free_pages.data_ptr(), free_pages.numel(),
                  free_count.data_ptr(), N, table.shape[1], int(page_size), *within, _lib.stream(lengths))


class _Like(NamedTuple):
    """A tensor's layout (_lib.layout) with as much of a tensor's face as the checks
    look at."""
    index: int
    dtype: torch.dtype
    shape: torch.Size
    strides: tuple

    is_cuda = property(lambda t: t.index >= 0)
    device = property(lambda t: torch.device("cuda", t.index) if t.index >= 0 else torch.device("cpu"))

    def dim(self):
        return len(self.shape)

    def numel(self):
        return math.prod(self.shape)

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def is_contiguous(self):
        expect = 1
        for size, stride in zip(reversed(self.shape), reversed(self.strides)):
            if size != 1 and stride != expect:
                return 0 in self.shape
            expect *= size
        return True


def _like(layout):
    return None if layout is None else _Like(*layout)


def _check_rows_of_slots(name, N, S, slots, rows):
    if slots.dtype != torch.int64 or slots.dim() != 2 or slots.shape[1] != S or (rows is None and slots.shape[0] != N):
        raise ValueError(f"{name}: slots must be int64 [{'R' if rows is not None else N}, {S}], got {slots.dtype} "
                         f"{tuple(slots.shape)}")
    if rows is not None:
        _vector(name, "rows", rows, torch.int64, N)


def store_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                slots: torch.Tensor, rows: Optional[torch.Tensor] = None, scales=None) -> None:
    """Writes the rows k, v [N, Hkv, S, hd] to their slots in the pool:
    prompt n's are `slots[n]`, or `slots[rows[n]]`, of int64 [R, S] (distinct;
    -1, or any outside the pool, for rows that are not kept).  rows: int64 [N],
    distinct; a row outside the slots stores nothing.  The pages are none of
    k's and v's memory.  Inference only: no gradient.

    `scales`: (k_scales, v_scales) of pages of 8 bits, which get the rows'
    scales.  int8: a row's largest value over 127 (at least 2^-126), e4m3: the
    least power of two that brings it to 448; values are rounded to nearest
    even.  A row with an infinity or NaN gets the scale NaN.  hd up to 256."""
    name = "store_pages"
    if scales is not None:
        _store_eight(name, k, v, k_pages, v_pages, slots, rows, scales)
        return
    _lib.require_gpu(name, k, v, k_pages, v_pages, slots, rows)
    check_pages(name, k_pages, v_pages)
    pages, K, page, hd = k_pages.shape
    if k.dim() != 4 or k.shape[1] != K or k.shape[3] != hd or v.shape != k.shape:
        raise ValueError(f"{name}: k and v must be [N, {K}, S, {hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    check_scales(name, k_pages, None, None)
    if not k.dtype == v.dtype == k_pages.dtype:
        raise ValueError(f"{name}: k, v and the pages must share a dtype")
    check_no_gradient(name, k, v, k_pages, v_pages)
    N, S = k.shape[0], k.shape[2]
    _check_rows_of_slots(name, N, S, slots, rows)
    k, v = (t if t.stride(-1) == 1 or hd == 1 else t.contiguous() for t in (k, v))
    slots, rows = slots.contiguous(), None if rows is None else rows.contiguous()
    with _lib.on_device(k):
        _lib.call("hydra_page_store", k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  slots.data_ptr(), slots.shape[0], _lib.ptr(rows), N, K, S, hd, pages, page, _strides(k), _strides(v),
                  _strides(k_pages), _strides(v_pages), _lib.dtype_code(k), _lib.stream(k))


@functools.lru_cache(maxsize=1024)
def _store_eight_call(name, *layouts):
    """The checks of a call of these layouts, once; what it is launched with beside
    addresses."""
    k, v, kp, vp, slots, rows, ks, vs = map(_like, layouts)
    _lib.require_gpu(name, k, v, kp, vp, slots, rows)
    check_pages(name, kp, vp)
    pages, K, page, hd = kp.shape
    if k.dim() != 4 or k.shape[1] != K or k.shape[3] != hd or v.shape != k.shape:
        raise ValueError(f"{name}: k and v must be [N, {K}, S, {hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    check_scales(name, kp, ks, vs)
    if k.dtype != v.dtype:
        raise ValueError(f"{name}: k and v must share a dtype")
    N, S = k.shape[0], k.shape[2]
    _check_rows_of_slots(name, N, S, slots, rows)
    # (without elements a copy would be the tensor itself, of whatever strides)
    copies = (N * S > 0 and hd > 1 and (k.stride(-1) != 1 or v.stride(-1) != 1)) or not slots.is_contiguous() or \
        not (rows is None or rows.is_contiguous())
    return (copies, slots.shape[0], (N, K, S, hd, pages, page, *map(_strides, (k, v, kp, vp, ks, vs)), _lib.dtype_code(k),
                                     _lib.PAGE_CODE[kp.dtype]), _lib.load().hydra_page_store8)


def _store_eight(name, k, v, k_pages, v_pages, slots, rows, scales):
    ks, vs = scales
    layout = _lib.layout
    copies, R, sizes, entry = _store_eight_call(name, layout(k), layout(v), layout(k_pages), layout(v_pages), layout(slots),
                                                layout(rows), layout(ks), layout(vs))
    check_no_gradient(name, k, v, k_pages, v_pages, ks, vs)
    if copies:
        _store_eight(name, k.contiguous(), v.contiguous(), k_pages, v_pages, slots.contiguous(),
                     None if rows is None else rows.contiguous(), scales)
        return
    with _lib.on_device(k):
        rc = entry(k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), ks.data_ptr(), vs.data_ptr(),
                   slots.data_ptr(), R, None if rows is None else rows.data_ptr(), *sizes, _lib.stream(k))
    _lib.check(rc, "hydra_page_store8")


@functools.lru_cache(maxsize=1024)
def _read_call(name, dtype, *layouts):
    """As _store_eight_call."""
    kp, vp, slots, rows, ks, vs = map(_like, layouts)
    _lib.require_gpu(name, kp, vp, slots, rows)
    check_pages(name, kp, vp)
    pages, K, page, hd = kp.shape
    check_scales(name, kp, ks, vs)
    if ks is None:
        if dtype not in (None, kp.dtype):
            raise ValueError(f"{name}: pages of {str(kp.dtype)[6:]} are read as they are, not as {str(dtype)[6:]}")
        dtype = kp.dtype
    elif dtype is None:
        raise ValueError(f"{name}: say which dtype (pages of {str(kp.dtype)[6:]})")
    if slots.dim() != 2 or (rows is not None and rows.dim() != 1):
        raise ValueError(f"{name}: slots must be int64 [N, S], got {slots.dtype} {tuple(slots.shape)}")
    N, S = (slots if rows is None else rows).shape[0], slots.shape[1]
    _check_rows_of_slots(name, N, S, slots, rows)
    shape = (N, K, S, hd)
    out = _Like(0, dtype, torch.Size(shape), (K * S * hd, S * hd, hd, 1))
    code = _lib.dtype_code(out)
    return (dtype, (2, *shape), (*shape, pages, page, _strides(kp), _strides(vp),
                                 *((None, None) if ks is None else (_strides(ks), _strides(vs))), _strides(out),
                                 _strides(out), code, code if ks is None else _lib.PAGE_CODE[kp.dtype]),
            _lib.load().hydra_page_read)


def read_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor,
               rows: Optional[torch.Tensor] = None, scales=None,
               dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """k, v [N, Hkv, S, hd] out of their slots, the way store_pages put them
    there: prompt n's are `slots[n]` of int64 [N, S], or `slots[rows[n]]`.  Zeros
    where a slot or a row is none.  Pages of 8 bits need their `scales` and the
    `dtype` wanted (bf16, fp16 or fp32; each value is rounded once); others
    are read as they are.  hd up to 256.  Inference only: no gradient."""
    name = "read_pages"
    ks, vs = (None, None) if scales is None else scales
    layout = _lib.layout
    dtype, shape, sizes, entry = _read_call(name, dtype, layout(k_pages), layout(v_pages), layout(slots), layout(rows),
                                            layout(ks), layout(vs))
    check_no_gradient(name, k_pages, v_pages, ks, vs)
    slots, rows = slots.contiguous(), None if rows is None else rows.contiguous()
    out = torch.empty(shape, dtype=dtype, device=k_pages.device)
    k, v = out.unbind(0)
    with _lib.on_device(k):
        rc = entry(k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(ks), _lib.ptr(vs), k.data_ptr(), v.data_ptr(),
                   slots.data_ptr(), slots.shape[0], _lib.ptr(rows), *sizes, _lib.stream(k))
    _lib.check(rc, "hydra_page_read")
    return k, v


def check_scales(name: str, pages, k_scales, v_scales) -> None:
    """Scales go with pages of 8 bits, and with no others."""
    eight = pages.dtype in _lib.PAGE_CODE
    if k_scales is None or v_scales is None:
        if eight:
            raise ValueError(f"{name}: pages of {str(pages.dtype)[6:]} need scales")
        return
    if not eight:
        raise ValueError(f"{name}: scales are of pages of 8 bits, these are {str(pages.dtype)[6:]}")
    _lib.require_gpu(name, pages, k_scales, v_scales)
    for t in (k_scales, v_scales):
        if t.dtype != torch.float32 or t.shape != pages.shape[:3]:
            raise ValueError(f"{name}: scales must be float32 {list(pages.shape[:3])}, got {t.dtype} {tuple(t.shape)}")
        if not t.is_contiguous():
            check_distinct(name, "scales", t)


@functools.lru_cache(maxsize=1024)
def _attention_workspace(device: int, *sizes) -> int:
    """Scratch bytes of these sizes on a device, which is current."""
    need = ctypes.c_int64(0)
    _lib.call("hydra_paged_attn_workspace", *sizes, ctypes.byref(need))
    return need.value


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    scales=None, shared: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q k^T) v of one query token per request, q [N, Hq, hd],
    over the first `lengths[i]` (int32) positions of its pages; query head h
    reads key head h // (Hq / Hkv).  scale: hd ** -0.5 by default.  `out`: a
    [N, Hq, hd] tensor with a unit last stride to write to (q itself is one;
    otherwise none of the memory that is read).

    `scales`: (k_scales, v_scales) of pages of 8 bits (store_pages).  `shared`:
    int32 [groups]; the N / groups requests from g N / groups on hold the same
    in their first shared[g] positions, which are read once for all of them,
    from the pages of the first one that is as long.  A request that is shorter
    is answered from its own pages alone.

    fp32 scores, softmax and sums, one rounding (with scales or shared a weight
    enters its product as two 16-bit terms, to 2^-16 of it, of fp16 pages to 2^-22
    of it and 2^-38 of the largest one, and an infinity among the values seen may
    come out as NaN; fp32 queries have fp32 weights).  Lengths count within
    [0, P * page_size]; keys on a page outside the pool are not seen; a
    request that sees none (or whose scores are all -inf) gets zeros.  Inference
    only: no gradient."""
    name = "paged_attention"
    if scales is not None or shared is not None:
        return _prefix_attention(name, q, k_pages, v_pages, table, lengths, None if scale is None else float(scale), out,
                                 scales, shared)
    _lib.require_gpu(name, q, k_pages, v_pages, table, lengths, out)
    check_pages(name, k_pages, v_pages)
    pages, K, page, hd = k_pages.shape
    if q.dim() != 3 or q.shape[2] != hd:
        raise ValueError(f"{name}: q must be [N, Hq, {hd}], got {tuple(q.shape)}")
    N, H, _ = q.shape
    if H == 0 or H % K != 0:
        raise ValueError(f"{name}: {H} query heads are no multiple of {K} key heads")
    check_scales(name, k_pages, None, None)
    if q.dtype != k_pages.dtype:
        raise ValueError(f"{name}: q and the pages must share a dtype")
    check_no_gradient(name, q, k_pages, v_pages, out)
    _vector(name, "lengths", lengths, torch.int32, N)
    _check_table(name, table, N)
    if table.shape[1] == 0:
        raise ValueError(f"{name}: a table without pages")
    if q.stride(-1) != 1 and hd > 1:
        q = q.contiguous()
    if out is None:
        out = q.new_empty((N, H, hd))
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError(f"{name}: out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif not out.is_contiguous():
        check_distinct(name, "rows of out", out)
    lengths = lengths.contiguous()
    P, code = table.shape[1], _lib.dtype_code(q)
    with _lib.on_device(q):
        need = _attention_workspace(q.device.index, N, H, K, hd, P, page, code)
        ws = _lib.scratch(need, q) if need else None
        _lib.call("hydra_paged_attn", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(),
                  table.data_ptr(), _row_stride(table), lengths.data_ptr(), N, H, K, hd, P, page, pages, _strides(q),
                  _strides(k_pages), _strides(v_pages), _strides(out), hd ** -0.5 if scale is None else float(scale),
                  code, _lib.ptr(ws), need, _lib.stream(q))
    return out


@functools.lru_cache(maxsize=1024)
def _prefix_call(name, scale, *layouts):
    """The checks of a call of these layouts, once; what it is launched with beside
    addresses, and the bytes of scratch.  On the tensors' device, which is current."""
    q, kp, vp, table, lengths, out, ks, vs, shared = map(_like, layouts)
    _lib.require_gpu(name, q, kp, vp, table, lengths, out, shared)
    check_pages(name, kp, vp)
    pages, K, page, hd = kp.shape
    if q.dim() != 3 or q.shape[2] != hd:
        raise ValueError(f"{name}: q must be [N, Hq, {hd}], got {tuple(q.shape)}")
    N, H, _ = q.shape
    if H == 0 or H % K != 0:
        raise ValueError(f"{name}: {H} query heads are no multiple of {K} key heads")
    check_scales(name, kp, ks, vs)
    if ks is None and q.dtype != kp.dtype:
        raise ValueError(f"{name}: q and the pages must share a dtype")
    _vector(name, "lengths", lengths, torch.int32, N)
    _check_table(name, table, N)
    if table.shape[1] == 0:
        raise ValueError(f"{name}: a table without pages")
    if out is None:
        out = q._replace(strides=(H * hd, hd, 1))
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError(f"{name}: out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif not out.is_contiguous():
        check_distinct(name, "rows of out", out)
    groups = 0
    if shared is not None:
        groups = _vector(name, "shared", shared, torch.int32).shape[0]
        if (groups == 0 and N > 0) or (groups > 0 and N % groups != 0):
            raise ValueError(f"{name}: {N} requests are no multiple of {groups} groups")
        if groups == N:  # nobody shares anything
            groups = 0
    P, code = table.shape[1], _lib.dtype_code(q)
    copies = (N > 0 and hd > 1 and q.stride(-1) != 1) or not lengths.is_contiguous() or \
        not (shared is None or shared.is_contiguous())  # (an empty q counts as contiguous whatever its strides)
    if groups == 0 and ks is None:
        return copies, None, 0, 0, None, None
    of = code if ks is None else _lib.PAGE_CODE[kp.dtype]
    need = ctypes.c_int64(0)
    _lib.call("hydra_prefix_attn_workspace", groups, N, H, K, hd, P, page, code, of, ctypes.byref(need))
    return (copies, (groups, N, H, K, hd, P, page, pages, _strides(q), _strides(kp), _strides(vp),
                     *((None, None) if ks is None else (_strides(ks), _strides(vs))), _strides(out),
                     hd ** -0.5 if scale is None else scale, code, of), groups, need.value, _row_stride(table),
            _lib.load().hydra_prefix_attn)


def _prefix_attention(name, q, k_pages, v_pages, table, lengths, scale, out, scales, shared):
    """paged_attention with scales, groups or both."""
    ks, vs = (None, None) if scales is None else scales
    layout = _lib.layout
    _lib.require_gpu(name, q)
    with _lib.on_device(q):
        copies, sizes, groups, need, table_rs, entry = _prefix_call(
            name, scale, layout(q), layout(k_pages), layout(v_pages), layout(table), layout(lengths), layout(out),
            layout(ks), layout(vs), layout(shared))
        check_no_gradient(name, q, k_pages, v_pages, out, ks, vs)
        if copies:
            return _prefix_attention(name, q.contiguous(), k_pages, v_pages, table, lengths.contiguous(), scale, out, scales,
                                     None if shared is None else shared.contiguous())
        if sizes is None:
            return paged_attention(q, k_pages, v_pages, table, lengths, scale, out)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ws = _lib.scratch(need, q) if need else None
        rc = entry(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), None if ks is None else ks.data_ptr(),
                   None if vs is None else vs.data_ptr(), out.data_ptr(), table.data_ptr(), table_rs, lengths.data_ptr(),
                   shared.data_ptr() if groups else None, *sizes, None if ws is None else ws.data_ptr(), need,
                   _lib.stream(q))
    _lib.check(rc, "hydra_prefix_attn")
    return out


class PageFork(NamedTuple):
    """What fork_pages did: `parents` int32 [N], the row that each row goes on
    from (-1: it holds nothing); `sources`, `copies` int32 [N], the page to copy
    for a row and where to (-1: none; copy_pages); `granted` bool [N]."""
    parents: torch.Tensor
    sources: torch.Tensor
    copies: torch.Tensor
    granted: torch.Tensor


@functools.lru_cache(maxsize=1024)
def _fork_call(name, *layouts):
    """The checks of a call of these layouts, once; what it is launched with beside
    addresses."""
    parents, lengths, table, free_pages, free_count, extra = map(_like, layouts)
    _lib.require_gpu(name, parents, lengths, table, free_pages, free_count, extra)
    N = _vector(name, "lengths", lengths, torch.int32).shape[0]
    _vector(name, "parents", parents, torch.int32, N)
    _vector(name, "free_pages", free_pages, torch.int32)
    _vector(name, "free_count", free_count, torch.int32, 1)
    pages = _vector(name, "extra", extra, torch.int32).shape[0]
    _check_table(name, table, N)
    P = table.shape[1]
    if N == 0 or P == 0 or pages == 0:
        raise ValueError(f"{name}: {N} rows of {P} pages in a pool of {pages}")
    _in_place(name, "lengths", lengths)
    _in_place(name, "free_pages", free_pages)
    _in_place(name, "extra", extra)
    need = ctypes.c_int64(0)
    _lib.call("hydra_page_fork_workspace", N, P, pages, ctypes.byref(need))
    return N, P, pages, need.value, _row_stride(table), free_pages.numel(), _lib.load().hydra_page_fork


def fork_pages(parents: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, extra: torch.Tensor, page_size: int) -> PageFork:
    """Row i goes on from what row parents[i] (int32 [N]; any outside [0, N):
    from nothing) held: its length, and its pages of `table`, all rows at once and
    in place.

    Pages that are full are held in common; `extra` (int32, one for each page of
    the pool) counts a page's holders beyond the first.  The page that a row was
    still filling stays with the first row that goes on from it; the others get
    copies, taken from the stack in their order, which copy_pages fills.  Pages that
    nobody holds any more go on the stack before that, in the order of rows and
    columns.  A row that finds no page for its copy is refused (`granted`) and
    holds nothing: where every row's last page is begun and each goes on from one
    of them, there are always enough.  At most 8192 rows."""
    name = "fork_pages"
    layout = _lib.layout
    N, P, pages, need, table_rs, stack, entry = _fork_call(name, layout(parents), layout(lengths), layout(table), layout(free_pages),
                                                    layout(free_count), layout(extra))
    parents = parents.contiguous()
    sources, copies, taken = lengths.new_empty((3, N)).unbind(0)
    granted = lengths.new_empty((N,), dtype=torch.bool)
    ws = _lib.scratch(need, lengths)
    with _lib.on_device(lengths):
        rc = entry(parents.data_ptr(), lengths.data_ptr(), table.data_ptr(), table_rs, free_pages.data_ptr(), stack,
                   free_count.data_ptr(), extra.data_ptr(), sources.data_ptr(), copies.data_ptr(), taken.data_ptr(),
                   granted.data_ptr(), N, P, int(page_size), pages, ws.data_ptr(), need, _lib.stream(lengths))
    _lib.check(rc, "hydra_page_fork")
    return PageFork(taken, sources, copies, granted)


@functools.lru_cache(maxsize=1024)
def _copy_call(name, *layouts):
    """As _fork_call."""
    kp, vp, sources, copies, ks, vs = map(_like, layouts)
    _lib.require_gpu(name, kp, vp, sources, copies)
    check_pages(name, kp, vp)
    pages, K, page, hd = kp.shape
    N = _vector(name, "sources", sources, torch.int32).shape[0]
    _vector(name, "copies", copies, torch.int32, N)
    check_scales(name, kp, ks, vs)
    if ks is None:
        _lib.dtype_code(kp)
    return ((N, K, hd, pages, page, _strides(kp), _strides(vp),
             *((None, None) if ks is None else (_strides(ks), _strides(vs))), kp.dtype.itemsize), _lib.load().hydra_page_copy)


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, sources: torch.Tensor, copies: torch.Tensor,
               scales=None) -> None:
    """Pages copies[i] become what pages sources[i] are (int32 [N]), in keys,
    values and `scales`.  Pairs with a page outside the pool are left out; copies
    are distinct and none is a source.  Inference only: no gradient."""
    name = "copy_pages"
    ks, vs = (None, None) if scales is None else scales
    layout = _lib.layout
    sizes, entry = _copy_call(name, layout(k_pages), layout(v_pages), layout(sources), layout(copies), layout(ks), layout(vs))
    check_no_gradient(name, k_pages, v_pages, ks, vs)
    sources, copies = sources.contiguous(), copies.contiguous()
    with _lib.on_device(k_pages):
        rc = entry(k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(ks), _lib.ptr(vs), sources.data_ptr(),
                   copies.data_ptr(), *sizes, _lib.stream(k_pages))
    _lib.check(rc, "hydra_page_copy")


@functools.lru_cache(maxsize=1024)
def _take_call(name, *layouts):
    """As _fork_call."""
    x, parents = map(_like, layouts)
    _lib.require_gpu(name, x, parents)
    if x.dim() == 0:
        raise ValueError(f"{name}: x must have rows")
    N = x.shape[0]
    _vector(name, "parents", parents, torch.int32, N)
    if x.numel() == 0:
        return 0, 0, 0, None
    row, e = x.numel() // N, x.dtype.itemsize
    inner = x._replace(shape=x.shape[1:], strides=x.strides[1:])
    if not inner.is_contiguous() or (N > 1 and x.stride(0) < row):
        raise ValueError(f"{name}: rows of strides {x.stride()} are not contiguous")
    return (x.stride(0) if N > 1 else row) * e, row * e, N, _lib.load().hydra_rows_take


def take_rows(x: torch.Tensor, parents: torch.Tensor) -> None:
    """x[i] = x[parents[i]] in place, all rows at once (int32 [N], N = len(x)
    up to 8192); a parent outside [0, N) leaves its row as it is.  Any dtype; rows
    are contiguous, do not overlap, and are none of the parents' memory.  Inference
    only: no gradient."""
    name = "take_rows"
    stride, row, N, entry = _take_call(name, _lib.layout(x), _lib.layout(parents))
    check_no_gradient(name, x)
    if N == 0:
        return
    parents = parents.contiguous()
    with _lib.on_device(x):
        rc = entry(x.data_ptr(), stride, row, parents.data_ptr(), N, _lib.stream(x))
    _lib.check(rc, "hydra_rows_take")


class PagePool:
    """The pages of up to `requests` requests of up to `max_length` tokens
    (whatever the page size: a plan refuses what goes past it): which pages each
    holds and which nobody does.  Layers keep their keys and values in pools of
    `pages` pages of their own and share this.

    `plan(new_tokens, width)` takes a step's pages and moves the lengths on;
    `release(done)` returns finished requests' pages.  With `sharing`,
    `fork(parents)` makes requests go on from what others hold, with the full
    pages in common (up to 8192 requests).  All of it runs on the device, on the
    current stream; a captured step replays with the lengths that it finds."""

    def __init__(self, requests: int, max_length: int, pages: int, page_size: int = 64, device="cuda",
                 sharing: bool = False):
        if requests < 1 or max_length < 1 or pages < 1:
            raise ValueError(f"PagePool: {requests} requests of up to {max_length} tokens in {pages} pages")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024, 2048, 4096):
            raise ValueError(f"PagePool: page_size {page_size} is no power of two in [16, 4096]")
        if sharing and requests > 8192:
            raise ValueError(f"PagePool: pages are shared among up to 8192 requests, not {requests}")
        self.requests, self.pages, self.page_size = int(requests), int(pages), int(page_size)
        self.max_length = int(max_length)
        self.lengths = torch.zeros(self.requests, dtype=torch.int32, device=device)
        self.table = torch.full((self.requests, -(-self.max_length // self.page_size)), -1, dtype=torch.int32,
                                device=device)
        self.free_pages = torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), self.pages, dtype=torch.int32, device=device)
        # a page's holders beyond the first, and every request as its own continuation
        self.extra = torch.zeros(self.pages, dtype=torch.int32, device=device) if sharing else None
        self._rows = torch.arange(self.requests, dtype=torch.int32, device=device) if sharing else None

    def plan(self, new_tokens: torch.Tensor, width: int = 1, from_empty: bool = False) -> PagePlan:
        """plan_pages of these requests, taken: the pool's lengths and free
        pages (`plan.lengths`, `plan.free_count`) are those after it."""
        width = int(width)
        in_place = _lib.query("hydra_page_plan_in_place", self.requests, width) == 1
        plan = _plan("PagePool.plan", self.lengths, new_tokens, self.table, self.free_pages, self.free_count,
                     self.page_size, width, from_empty, self.max_length, in_place)
        if not in_place:
            self.lengths.copy_(plan.lengths)
            self.free_count.copy_(plan.free_count)
            plan = plan._replace(lengths=self.lengths, free_count=self.free_count)
        return plan

    def fork(self, parents: torch.Tensor) -> PageFork:
        """fork_pages of these requests: request i goes on from what request
        parents[i] holds.  Every layer's cache follows (CCGQACache.fork)."""
        if self.extra is None:
            raise RuntimeError("PagePool.fork: the pool shares no pages (sharing=True)")
        return fork_pages(parents, self.lengths, self.table, self.free_pages, self.free_count, self.extra,
                          self.page_size)

    def release(self, done: torch.Tensor) -> None:
        if self.extra is not None:  # a page comes back with its last holder
            _vector("PagePool.release", "done", done, torch.bool, self.requests)
            _lib.require_gpu("PagePool.release", done, self.lengths)
            self.fork(torch.where(done, -1, self._rows))
            return
        release_pages(done, self.lengths, self.table, self.free_pages, self.free_count, self.page_size, self.pages)
