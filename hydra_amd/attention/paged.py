"""A paged key-value cache: page tables planned on the GPU, key and value rows
stored into their pages, and the attention of one new token per request over
them.

A pool holds `k_pages` and `v_pages` [pages, Hkv, page_size, hd] (any strides
with a unit last one); position t of request i lies in page
`table[i, t // page_size]` at row `t % page_size`, and its *slot* is
`page * page_size + row`.  `page_size` is a power of two in [16, 4096].

Nothing here synchronises with the host, so what only the device knows is
settled there: a request that finds no room is refused by the plan
(`granted`), a slot or table entry outside the pool stores and shows nothing.

The reference has no cache (it recomputes the sequence for every token).
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

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


def store_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                slots: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
    """Writes the rows k, v [N, Hkv, S, hd] to their slots in the pool:
    prompt n's are `slots[n]`, or `slots[rows[n]]`, of int64 [R, S] (distinct;
    -1, or any outside the pool, for rows that are not kept).  rows: int64 [N],
    distinct; a row outside the slots stores nothing.  The pages are none of
    k's and v's memory.  Inference only: no gradient."""
    name = "store_pages"
    _lib.require_gpu(name, k, v, k_pages, v_pages, slots, rows)
    check_pages(name, k_pages, v_pages)
    pages, K, page, hd = k_pages.shape
    if k.dim() != 4 or k.shape[1] != K or k.shape[3] != hd or v.shape != k.shape:
        raise ValueError(f"{name}: k and v must be [N, {K}, S, {hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if not k.dtype == v.dtype == k_pages.dtype:
        raise ValueError(f"{name}: k, v and the pages must share a dtype")
    check_no_gradient(name, k, v, k_pages, v_pages)
    N, S = k.shape[0], k.shape[2]
    if slots.dtype != torch.int64 or slots.dim() != 2 or slots.shape[1] != S or (rows is None and slots.shape[0] != N):
        raise ValueError(f"{name}: slots must be int64 [{'R' if rows is not None else N}, {S}], got {slots.dtype} "
                         f"{tuple(slots.shape)}")
    if rows is not None:
        rows = _vector(name, "rows", rows, torch.int64, N).contiguous()
    k, v = (t if t.stride(-1) == 1 or hd == 1 else t.contiguous() for t in (k, v))
    slots = slots.contiguous()
    with _lib.on_device(k):
        _lib.call("hydra_page_store", k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  slots.data_ptr(), slots.shape[0], _lib.ptr(rows), N, K, S, hd, pages, page, _strides(k), _strides(v),
                  _strides(k_pages), _strides(v_pages), _lib.dtype_code(k), _lib.stream(k))


@functools.lru_cache(maxsize=1024)
def _attention_workspace(device: int, *sizes) -> int:
    """Scratch bytes of these sizes on a device, which is current."""
    need = ctypes.c_int64(0)
    _lib.call("hydra_paged_attn_workspace", *sizes, ctypes.byref(need))
    return need.value


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q k^T) v of one query token per request, q [N, Hq, hd],
    over the first `lengths[i]` (int32) positions of its pages; query head h
    reads key head h // (Hq / Hkv).  scale: hd ** -0.5 by default.  `out`: a
    [N, Hq, hd] tensor with a unit last stride to write to (q itself is one;
    otherwise none of the memory that is read).

    fp32 scores, softmax and sums, one rounding.  Lengths count within
    [0, P * page_size]; keys on a page outside the pool are not seen; a
    request that sees none (or whose scores are all -inf) gets zeros.  Inference
    only: no gradient."""
    name = "paged_attention"
    _lib.require_gpu(name, q, k_pages, v_pages, table, lengths, out)
    check_pages(name, k_pages, v_pages)
    pages, K, page, hd = k_pages.shape
    if q.dim() != 3 or q.shape[2] != hd:
        raise ValueError(f"{name}: q must be [N, Hq, {hd}], got {tuple(q.shape)}")
    N, H, _ = q.shape
    if H == 0 or H % K != 0:
        raise ValueError(f"{name}: {H} query heads are no multiple of {K} key heads")
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


class PagePool:
    """The pages of up to `requests` requests of up to `max_length` tokens
    (whatever the page size: a plan refuses what goes past it): which pages each
    holds and which nobody does.  Layers keep their keys and values in pools of
    `pages` pages of their own and share this.

    `plan(new_tokens, width)` takes a step's pages and moves the lengths on;
    `release(done)` returns finished requests' pages.  All of it runs on the
    device, on the current stream; a captured step replays with the lengths
    that it finds."""

    def __init__(self, requests: int, max_length: int, pages: int, page_size: int = 64, device="cuda"):
        if requests < 1 or max_length < 1 or pages < 1:
            raise ValueError(f"PagePool: {requests} requests of up to {max_length} tokens in {pages} pages")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024, 2048, 4096):
            raise ValueError(f"PagePool: page_size {page_size} is no power of two in [16, 4096]")
        self.requests, self.pages, self.page_size = int(requests), int(pages), int(page_size)
        self.max_length = int(max_length)
        self.lengths = torch.zeros(self.requests, dtype=torch.int32, device=device)
        self.table = torch.full((self.requests, -(-self.max_length // self.page_size)), -1, dtype=torch.int32,
                                device=device)
        self.free_pages = torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), self.pages, dtype=torch.int32, device=device)

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

    def release(self, done: torch.Tensor) -> None:
        release_pages(done, self.lengths, self.table, self.free_pages, self.free_count, self.page_size, self.pages)
