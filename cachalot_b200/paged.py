"""The decode step around the experts: page plan, query and key preparation, attention over a paged key-value cache,
log probabilities of the head's logits.

A cache of one layer is two tensors `k_cache` and `v_cache` [pages, kv_heads, page_size, head_dim] of float16, bfloat16 or
float8_e4m3fn (with one float32 scale per head: value = code * scale); other orders of the first three axes are views of
their own storage (`.transpose(1, 2)` of [pages, page_size, kv_heads, head_dim]).  A request's row of the block table
names its pages in order; slot = page * page_size + place within the page.

Lengths, positions, slots and ids are int32; int64 ones are narrowed (values beyond int32 become its largest or smallest).

Every function here calls the C ABI; as in `ops`, calls whose arguments already have the dtype and layout the kernels take
go through the native call path, and none has a PyTorch or CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import math
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
    """An int32 contiguous tensor of this shape.  int64 is narrowed, with values beyond int32 held at its ends: too long, past the
    cache or past the vocabulary as before, which wrapped they might not be."""
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    return (t.clamp(-2 ** 31, 2 ** 31 - 1) if t.dtype == torch.int64 else t).to(torch.int32).contiguous()


def _status(t: torch.Tensor | None) -> None:
    if t is not None and (t.dtype != torch.int32 or t.numel() < 1 or not t.is_contiguous()):
        raise ValueError("status must be an int32 word")


def _block_table(t: torch.Tensor, rows: int) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"block_table must be int32 [{rows}, width], got {t.dtype} {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("block_table rows must be contiguous")


_DT = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32, torch.float8_e4m3fn: _lib.E4M3}  # of the C ABI


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale, v_scale) -> _lib.PagedKV:
    """The descriptor of a cache of one layer."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache must both be [pages, kv_heads, page_size, head_dim], got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if k_cache.dtype != v_cache.dtype or k_cache.dtype not in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
        raise ValueError(f"a cache holds float16, bfloat16 or float8_e4m3fn, got {k_cache.dtype} and {v_cache.dtype}")
    pages, heads, page, dim = k_cache.shape
    for t in (k_cache, v_cache):
        if t.stride(3) != 1 and dim > 1:
            raise ValueError("the last axis of a cache must be contiguous")
    scaled = k_cache.dtype == torch.float8_e4m3fn
    for t in (k_scale, v_scale):
        if t is not None and (not scaled or t.dtype != torch.float32 or tuple(t.shape) != (heads,) or not t.is_contiguous()):
            raise ValueError(f"scales are float32 [{heads}] and belong to a float8_e4m3fn cache")
    d = _lib.PagedKV()
    d.k, d.v, d.k_scale, d.v_scale = _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale)
    d.k_page_stride, d.k_head_stride, d.k_token_stride = k_cache.stride()[:3]
    d.v_page_stride, d.v_head_stride, d.v_token_stride = v_cache.stride()[:3]
    d.n_pages, d.page_size, d.kv_heads, d.head_dim, d.dtype = pages, page, heads, dim, _DT[k_cache.dtype]
    return d


# ---- page plan --------------------------------------------------------------------------------

class PagePlan(NamedTuple):
    """Where a step's new tokens go: `starts` int32 [requests+1], per token `requests`, `positions`, `slots` int32 [tokens]
    (past the last one: -1, 0, -1), `lens` int32 [requests] with the new tokens, `free_count` int32 [1] pages left.

    They may be views of one allocation that do not overlap, as those of `torch.split`: any of them keeps all of it alive (clone
    what is kept longer than the step), and none may be resized, which would grow it over its neighbours."""

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
        return PagePlan._make(p)
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


# ---- queries and keys -------------------------------------------------------------------------

def rope_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0, trained_len: int = 0,
                     beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary_dim/2] in radians per position, magnitude) for `qk_norm_rope`, computed once on the host.
    f_i = base ** (-2i / rotary_dim).  For contexts `factor` times as long as the trained one: "linear" stretches every
    frequency, "ntk" raises the base so that the slowest one is stretched and the fastest kept, "yarn" (Peng et al. 2023)
    stretches those that turn less than beta_slow times over `trained_len` positions, keeps those that turn more than
    beta_fast times, blends in between and lengthens the rotated vector by 0.1 ln(factor) + 1."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if factor < 1.0 or base <= 1.0:
        raise ValueError(f"factor must be at least 1 and base above 1, got {factor} and {base}")
    magnitude = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        if trained_len <= 0:
            raise ValueError("yarn needs trained_len")
        pair = lambda turns: rotary_dim * math.log(trained_len / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rotary_dim - 1)
        stretched = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(rotary_dim // 2)]
        f = [x * (1.0 - s) + x / factor * s for x, s in zip(f, stretched)]
        magnitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(f, dtype=torch.float64, device=device), magnitude


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself if its heads are 16-byte rows, else a contiguous copy."""
    ok = t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False, magnitude: float = 1.0,
                 v: torch.Tensor | None = None, k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                 slots: torch.Tensor | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                 status: torch.Tensor | None = None):
    """Norm of every query and key head, position rotation and cache write of new tokens in one launch
    (model/norm_rope_mlx.py, model/decode_fused_metal.py:43): q [tokens, heads, dim], k and v [tokens, kv_heads, dim]
    float16 or bfloat16 (views of the projection's rows as they are), positions int32 [tokens].

    q_weight, k_weight [dim] (None: no norm); `inv_freq` and `magnitude` from `rope_frequencies`, the first
    2 * len(inv_freq) elements of a head are rotated, as pairs (i, i + half) or, `interleaved`, (2i, 2i + 1).  Everything
    in fp32 (angles in 64 bits), rounded once.  With a cache, keys and values go to `slots` int32 [tokens] (-1: not
    stored; a slot named twice in a call: undefined) and (q_out, None) is returned, else (q_out, k_out)."""
    r = _host.qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, magnitude, v, k_cache, v_cache, slots, k_scale, v_scale, status)
    if r is not None:
        return r
    dev = _same_device(q, k, positions, inv_freq, q_weight, k_weight, v, k_cache, v_cache, slots, k_scale, v_scale, status)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q and k must be [tokens, heads, dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype:
        raise ValueError(f"q and k must both be float16 or both bfloat16, got {q.dtype} and {k.dtype}")
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    pos = _ints(positions, "positions", (tokens,))
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1:
        raise ValueError(f"inv_freq must be float64 [rotary_dim / 2], got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    w_dtype = None
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            if tuple(w.shape) != (dim,) or w.dtype not in (q.dtype, torch.float32) or w_dtype not in (None, w.dtype):
                raise ValueError(f"{name} must be [{dim}] in {q.dtype} or float32 (both weights alike), got {w.dtype} {tuple(w.shape)}")
            w_dtype = w.dtype
    _status(status)
    desc = None
    with torch.cuda.device(dev):
        if k_cache is not None or v_cache is not None:
            if k_cache is None or v_cache is None or v is None or slots is None:
                raise ValueError("a cache write needs v, k_cache, v_cache and slots")
            if v.dtype != q.dtype or v.shape != k.shape:
                raise ValueError(f"v must be {q.dtype} {tuple(k.shape)}, got {v.dtype} {tuple(v.shape)}")
            desc = _cache(k_cache, v_cache, k_scale, v_scale)
            slots, v = _ints(slots, "slots", (tokens,)), _rows16(v)
        elif v is not None or slots is not None or k_scale is not None or v_scale is not None:
            raise ValueError("v, slots and scales go with k_cache and v_cache")
        q, k, inv_freq = _rows16(q), _rows16(k), inv_freq.contiguous()
        q_weight, k_weight = (None if w is None else w.contiguous().clone() if w.data_ptr() % 16 else w.contiguous() for w in (q_weight, k_weight))
        q_out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=dev)
        k_out = torch.empty((tokens, kv_heads, dim), dtype=q.dtype, device=dev) if desc is None else None
        check(lib.cachalot_qk_norm_rope(_ptr(q), q.stride(0), q.stride(1), _ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0) if v is not None else 0,
                                        v.stride(1) if v is not None else 0, _DT[q.dtype], tokens, heads, kv_heads, dim, _ptr(q_weight), _ptr(k_weight),
                                        _DT[w_dtype] if w_dtype is not None else _DT[q.dtype], eps, _ptr(pos), _ptr(inv_freq), 2 * inv_freq.numel(),
                                        int(interleaved), magnitude, _ptr(q_out), _ptr(k_out), None if desc is None else C.byref(desc), _ptr(slots),
                                        _ptr(status), _stream(dev)))
    return q_out, k_out


# ---- attention --------------------------------------------------------------------------------

def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, *,
                    scale: float | None = None, window: int = 0, softcap: float = 0.0, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, want_lse: bool = False,
                    status: torch.Tensor | None = None):
    """One new token per request over its pages (grouped-query decode attention, minimax/gqa_decode.py:180-187):
    q [requests, heads, dim] float16 or bfloat16, caches as `qk_norm_rope` fills them, block_table int32 [requests, width],
    lens int32 [requests] = visible tokens, the new one among them.  Query head i reads key-value head
    i // (heads // kv_heads); `scale` defaults to dim ** -0.5; softcap > 0: scores softcap * tanh(s / softcap); window > 0:
    only the last `window` tokens.  Returns out [requests, heads, dim] in `out_dtype` (default: q's), with `want_lse` also
    float32 [requests, heads] log sum exp of the scores.  Scores and sums are float32; softmax weights meet the values with 16
    bits over a bfloat16 cache, 22 over a float16 one, and over an E4M3 one 11 for bfloat16 results, 22 for others.  A request of length 0
    gives zeros and -inf; tokens whose table entry is no page of the cache are hidden, lengths past the table cut (bits in
    `status`).  The lengths are read on the device: nothing waits for them, and a captured call replays with new ones.  What
    suits many short requests (up to 1024 tokens, 4096 over E4M3) is chosen by how many tokens a row of `block_table` holds, or by the
    window: a view of the table's first columns that the batch needs makes such a batch up to twice as fast."""
    r = _host.paged_attention(q, k_cache, v_cache, block_table, lens, scale, window, softcap, k_scale, v_scale,
                              None if out_dtype is None else _DT.get(out_dtype, -1), want_lse, status)
    if r is not None:
        return r
    dev = _same_device(q, k_cache, v_cache, block_table, lens, k_scale, v_scale, status)
    if q.dim() != 3:
        raise ValueError(f"q must be [requests, heads, dim], got {tuple(q.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q must be float16 or bfloat16, got {q.dtype}")
    out_dtype = q.dtype if out_dtype is None else out_dtype
    if out_dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError(f"out_dtype must be float16, bfloat16 or float32, got {out_dtype}")
    requests, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    desc = _cache(k_cache, v_cache, k_scale, v_scale)
    if desc.head_dim != dim:
        raise ValueError(f"q has heads of {dim}, the cache of {desc.head_dim}")
    _block_table(block_table, requests)
    n = _ints(lens, "lens", (requests,))
    _status(status)
    if not 0 <= window < 2 ** 31:
        raise ValueError(f"window must be in [0, 2**31), got {window}")
    with torch.cuda.device(dev):
        if q.stride(2) != 1 or q.stride(0) % 2 or q.stride(1) % 2 or q.data_ptr() % 4:
            q = q.clone(memory_format=torch.contiguous_format)
        out = torch.empty((requests, heads, dim), dtype=out_dtype, device=dev)
        lse = torch.empty((requests, heads), dtype=torch.float32, device=dev) if want_lse else None
        need = lib.cachalot_paged_attention_workspace_bytes(heads, desc.kv_heads, dim, desc.dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)  # of this call: a captured graph keeps its own
        check(lib.cachalot_paged_attention(_ptr(q), q.stride(0), q.stride(1), _DT[q.dtype], requests, heads, C.byref(desc), _ptr(block_table),
                                           block_table.stride(0), block_table.shape[1], _ptr(n), scale, window, softcap, _ptr(ws), need, _ptr(out),
                                           _DT[out_dtype], _ptr(lse), _ptr(status), _stream(dev)))
    return (out, lse) if want_lse else out


# ---- log probabilities ------------------------------------------------------------------------

class TokenLogprobs(NamedTuple):
    """float32 `logprobs` and `entropy` [rows], `top_ids` int32 and `top_logprobs` float32 [rows, top]; views of one allocation as those
    of `PagePlan`."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, status: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probability of tokens int32 [rows] under logits [rows, vocab] (float32 as `bf16_gemv_f32` gives them, bfloat16 or
    float16), entropy of each row in nats and the `top` <= 32 most likely tokens (ties to the lower index), in one pass over
    the logits.  A negative id is padding (log probability 0), as is one past the vocabulary (STATUS_ID_RANGE); logits
    of -inf have no weight, and a row of nothing else gives -inf and entropy 0."""
    r = _host.token_logprobs(logits, tokens, top, status)
    if r is not None:
        return TokenLogprobs._make(r)
    dev = _same_device(logits, tokens, status)
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"logits must be float32, bfloat16 or float16 [rows, vocab], got {logits.dtype} {tuple(logits.shape)}")
    rows, vocab = logits.shape
    ids = _ints(tokens, "tokens", (rows,))
    _status(status)
    if not 0 <= top < 2 ** 31:
        raise ValueError(f"top must be in [0, 32], got {top}")
    with torch.cuda.device(dev):
        x = logits if logits.stride(1) == 1 else logits.contiguous()
        logprobs, entropy = (torch.empty(rows, dtype=torch.float32, device=dev) for _ in range(2))
        top_ids, top_logprobs = (torch.empty((rows, min(top, vocab)), dtype=t, device=dev) for t in (torch.int32, torch.float32))
        check(lib.cachalot_token_logprobs(_ptr(x), _DT[x.dtype], x.stride(0), rows, vocab, _ptr(ids), top, _ptr(logprobs), _ptr(entropy), _ptr(top_ids),
                                          _ptr(top_logprobs), _ptr(status), _stream(dev)))
    return TokenLogprobs(logprobs, entropy, top_ids, top_logprobs)
