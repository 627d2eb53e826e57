"""The decode step around the experts: page plan, query and key preparation, attention over a paged key-value cache.

A cache of one layer is two tensors `k_cache` and `v_cache` [pages, kv_heads, page_size, head_dim] of float16, bfloat16 or
float8_e4m3fn (with one float32 scale per head: value = code * scale); other orders of the first three axes are views of
their own storage (`.transpose(1, 2)` of [pages, page_size, kv_heads, head_dim]).  A request's row of the block table
names its pages in order; slot = page * page_size + place within the page.

Every function here calls the C ABI; as in `ops`, calls whose arguments already have the dtype and layout the kernels take
go through the native call path, and none has a PyTorch or CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib
from .ops import _host, _need_cuda, _ptr


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _same_device(*ts) -> torch.device:
    _need_cuda(*ts)
    devices = {t.device for t in ts if t is not None}
    if len(devices) != 1:
        raise ValueError(f"tensors on different devices: {sorted(map(str, devices))}")
    return devices.pop()


def _ints(t: torch.Tensor, name: str, shape: tuple) -> torch.Tensor:
    """An int32 contiguous tensor of this shape (int64 is narrowed)."""
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    return t.to(torch.int32).contiguous()


def _status(t: torch.Tensor | None) -> None:
    if t is not None and (t.dtype != torch.int32 or t.numel() < 1 or not t.is_contiguous()):
        raise ValueError("status must be an int32 word")


def _block_table(t: torch.Tensor, rows: int) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"block_table must be int32 [{rows}, width], got {t.dtype} {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("block_table rows must be contiguous")


# ---- page plan --------------------------------------------------------------------------------

class PagePlan(NamedTuple):
    """Where a step's new tokens go: `starts` int32 [requests+1], per token `requests`, `positions`, `slots` int32 [tokens]
    (past the last one: -1, 0, -1), `lens` int32 [requests] with the new tokens, `free_count` int32 [1] pages left."""

    starts: torch.Tensor
    requests: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    lens: torch.Tensor
    free_count: torch.Tensor


def plan_pages(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, *, page_size: int, tokens: int, status: torch.Tensor | None = None) -> PagePlan:
    """Block tables and slots of a step's new tokens in one launch, from lengths on the device (no host round trip):
    request r holds context_lens[r] tokens and gets new_lens[r] more.  Pages come from the end of
    free_pages[:free_count], request by request, and are written into `block_table` (int32 [requests, width], in place;
    entries that no new page goes to stay as they are).  `tokens` is the size of the step, e.g. that of a captured
    graph: new tokens beyond it are left out as if not asked for.  Tokens that get no page have slot -1; `status`
    (int32 word) gets STATUS_NO_PAGE or STATUS_LENGTH.  `free_pages` itself is not changed: the next call gets the plan's
    `free_count`, and pages given back are appended at that place."""
    p = _host.plan_pages(context_lens, new_lens, block_table, free_pages, free_count, page_size, tokens, status)
    if p is not None:
        return PagePlan(*p)
    dev = _same_device(context_lens, new_lens, block_table, free_pages, free_count, status)
    r = context_lens.numel()
    ctx, new = _ints(context_lens, "context_lens", (r,)), _ints(new_lens, "new_lens", (r,))
    _block_table(block_table, r)
    free = _ints(free_pages, "free_pages", (free_pages.numel(),))
    if free_count.numel() != 1:
        raise ValueError(f"free_count must be one number, got {tuple(free_count.shape)}")
    count = _ints(free_count.reshape(1), "free_count", (1,))
    _status(status)
    if not 0 <= tokens < 2 ** 31:
        raise ValueError(f"tokens must be in [0, 2**31), got {tokens}")
    if not 0 < page_size < 2 ** 31:
        raise ValueError(f"page_size must be positive, got {page_size}")
    with torch.cuda.device(dev):
        starts, requests, positions, slots, lens, left = (torch.empty(n, dtype=torch.int32, device=dev) for n in (r + 1, tokens, tokens, tokens, r, 1))
        check(lib.cachalot_plan_pages(_ptr(ctx), _ptr(new), r, _ptr(block_table), block_table.stride(0), block_table.shape[1], _ptr(free), free.numel(),
                                      _ptr(count), page_size, tokens, _ptr(starts), _ptr(requests), _ptr(positions), _ptr(slots), _ptr(lens),
                                      _ptr(left), _ptr(status), _stream(dev)))
    return PagePlan(starts, requests, positions, slots, lens, left)
