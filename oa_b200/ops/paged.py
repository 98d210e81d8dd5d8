"""A key-value cache in pages for requests of unequal length, on raw tensors: page tables and slot maps, rotary append, attention behind a
shared prompt.

Layout contract: the cache of a layer is a pair [pages, kv_heads, page_size, head_dim] (16, 32, 64 or 128 tokens a page; the stride between
pages is free, so that keys and values may lie in one tensor).  A request owns the pages in its row of `tables` [batch, width] int32, the
slot of a token is page * page_size + offset, and `free_pages` is a stack of which the first `taken` entries are in use.  The prompt that
all requests share has pages of its own, in a table of its own; lengths count a request's own tokens without it.

CUDA tensors run csrc/kernels/paged.cu and paged_attn.cu; CPU tensors the plain statement of the same mathematics.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import torch

from .. import _native as N
from . import kernels as K

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128)       # of the attention kernels; the CPU path takes any


class PagedStep(NamedTuple):
    """What a step of a batch needs to know about its tokens (int32, on the requests' device)."""
    starts: torch.Tensor        # [batch + 1] first token of each request
    lens: torch.Tensor          # [batch] own tokens of each request after the step
    slots: torch.Tensor         # [tokens] where a token's key and value go; -1: nowhere
    positions: torch.Tensor     # [tokens] position of a token, position0 included; -1 beyond the step's tokens
    rows: torch.Tensor          # [tokens] request of a token; -1 beyond the step's tokens
    taken: torch.Tensor         # [1] pages of the stack in use after the step
    missing: torch.Tensor       # [1] tokens without a slot (no page left, or the table's row full), plus those beyond `tokens`


_I32 = torch.int32


def _int32(what: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype is not _I32 or not t.is_contiguous():
            raise ValueError(f"{what}: contiguous int32 tensors expected")


def _table(what: str, tables: torch.Tensor, batch: int):
    """(width, elements between rows) of a table of `batch` rows."""
    return _table_layout(what, tables.shape, tables.stride(), tables.dtype, batch)


def _table_layout(what: str, shape, stride, dtype, batch: int):
    if dtype is not _I32 or len(shape) != 2:
        raise ValueError(f"{what}: tables must be int32 [{batch}, width]")
    rows, width = shape
    step, unit = stride
    if rows != batch or (width > 1 and unit != 1) or (batch > 1 and step < width):
        raise ValueError(f"{what}: tables must be int32 [{batch}, width] with rows side by side")
    return width, step if batch > 1 else width


def _same_device(what: str, first: torch.Tensor, *tensors: torch.Tensor) -> None:
    at = first.get_device()
    for t in tensors:
        if t.get_device() != at:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def _aligned_rows(t: torch.Tensor, rows: int, cols: int):
    """(the rows as the kernels read them, elements between rows): elements side by side, every row on 16 bytes.  A copy where they are not."""
    step, unit = t.stride()
    if rows <= 1:
        step = cols                                  # the stride of a single row says nothing
    if unit == 1 and step * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0:
        return t, step
    return (t.clone(memory_format=torch.contiguous_format) if t.is_contiguous() else K.contiguous(t)), cols


def plan(cached: torch.Tensor, fresh: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor, page_size: int,
         tokens: int, position0: int = 0) -> PagedStep:
    """Room for `fresh` [batch] new tokens of requests that hold `cached` [batch]: pages go from the stack into `tables` (in place), tokens lie
    one request after the other.  `tokens` is the number of token rows the caller has (rows beyond the step's are marked -1); `position0` the
    length of what all requests share.  Nothing is read back to the host; `taken` is not changed, the step holds the new one.  Lengths
    are not negative and sum up below 2^31."""
    batch = cached.numel()
    if page_size not in PAGE_SIZES:
        raise ValueError(f"plan: a page holds one of {PAGE_SIZES} tokens, not {page_size}")
    if fresh.numel() != batch or taken.numel() != 1 or tokens < 0:
        raise ValueError("plan: cached and fresh of one batch, taken of one number, tokens not negative")
    _int32("plan", cached, fresh, free_pages, taken)
    width, row_stride = _table("plan", tables, batch)
    _same_device("plan", cached, fresh, tables, free_pages, taken)
    if not cached.is_cuda:
        return _plan_cpu(cached, fresh, tables, free_pages, taken, page_size, tokens, position0)
    out = torch.empty(2 * batch + 3 * tokens + 3, dtype=torch.int32, device=cached.device)
    a = out.data_ptr()
    b = a + 4 * (2 * batch + 1)
    K._launch(N.require().oa_paged_plan(cached.data_ptr(), fresh.data_ptr(), tables.data_ptr(), row_stride, free_pages.data_ptr(), taken.data_ptr(),
                                        a, a + 4 * (batch + 1), b, b + 4 * tokens, b + 8 * tokens, b + 12 * tokens, b + 12 * tokens + 4, batch, width,
                                        free_pages.numel(), page_size, tokens, position0, N.stream()), "oa_paged_plan")
    return PagedStep._make(torch.unsafe_split_with_sizes(out, (batch + 1, batch, tokens, tokens, tokens, 1, 1)))


def _plan_cpu(cached, fresh, tables, free_pages, taken, ps, tokens, position0) -> PagedStep:
    width, n_free = tables.shape[1], free_pages.numel()
    top = min(max(int(taken), 0), n_free)
    starts, lens, slots, positions, rows, missing = [0], [], [], [], [], 0
    for b, (c, f) in enumerate(zip(cached.clamp(min=0).tolist(), fresh.clamp(min=0).tolist())):
        for j in range(min(-(-c // ps), width), min(-(-(c + f) // ps), width)):
            tables[b, j] = free_pages[top] if top < n_free else -1
            top = min(top + 1, n_free)
        for at in range(c, c + f):
            page = int(tables[b, at // ps]) if at // ps < width else -1
            slots.append(page * ps + at % ps if page >= 0 else -1)
            missing += page < 0
            positions.append(at + position0)
            rows.append(b)
        starts.append(starts[-1] + f)
        lens.append(min(c + f, width * ps))

    def ints(v, n=None):
        return torch.tensor(v if n is None else (v + [-1] * n)[:n], dtype=torch.int32)

    return PagedStep(ints(starts), ints(lens), ints(slots, tokens), ints(positions, tokens), ints(rows, tokens), ints([top]),
                     ints([missing + max(0, starts[-1] - tokens)]))


def release(done: torch.Tensor, lens: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor, page_size: int) -> torch.Tensor:
    """Puts the pages of the requests marked in `done` [batch] (bool) back on the stack: their lengths become 0 and their table entries -1, in
    place; returns the new `taken`."""
    batch = lens.numel()
    if page_size not in PAGE_SIZES:
        raise ValueError(f"release: a page holds one of {PAGE_SIZES} tokens, not {page_size}")
    if done.dtype != torch.bool or done.numel() != batch or not done.is_contiguous() or taken.numel() != 1:
        raise ValueError("release: done must be a contiguous bool tensor with one entry for each request, taken one number")
    _int32("release", lens, free_pages, taken)
    width, row_stride = _table("release", tables, batch)
    _same_device("release", lens, done, tables, free_pages, taken)
    if not lens.is_cuda:
        top = min(max(int(taken), 0), free_pages.numel())
        for b in range(batch):
            if done[b]:
                n = min(-(-max(int(lens[b]), 0) // page_size), width)
                pages = [int(i) for i in tables[b, :n] if i >= 0]
                back = top - len(pages)
                for k, i in enumerate(pages):
                    if back + k >= 0:
                        free_pages[back + k] = i
                top = max(back, 0)
                tables[b, :n] = -1
                lens[b] = 0
        return torch.tensor([top], dtype=torch.int32)
    now = torch.empty(1, dtype=torch.int32, device=lens.device)
    K._launch(N.require().oa_paged_release(done.data_ptr(), lens.data_ptr(), tables.data_ptr(), row_stride, free_pages.data_ptr(),
                                           free_pages.numel(), taken.data_ptr(), now.data_ptr(), batch, width, page_size, N.stream()),
              "oa_paged_release")
    return now


# What follows from shapes, strides and types alone is worked out once for each of them: a step makes these calls for every layer, and the checks
# took longer than the launch.
@functools.lru_cache(maxsize=256)
def _pool(what: str, shape, k_stride, v_shape, v_stride, k_dtype, v_dtype, dtype: torch.dtype):
    """(pages, kv heads, page size, head dim, elements between pages of k, and of v) of a pool."""
    if len(shape) != 4 or shape != v_shape or k_dtype is not dtype or v_dtype is not dtype:
        raise ValueError(f"{what}: k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] of {dtype}")
    pages, heads, ps, hd = shape
    if ps not in PAGE_SIZES:
        raise ValueError(f"{what}: a page holds one of {PAGE_SIZES} tokens, not {ps}")
    k0, *k_in = k_stride
    v0, *v_in = v_stride
    if k_in != [ps * hd, hd, 1] or v_in != k_in or (pages > 1 and min(k0, v0) < heads * ps * hd):
        raise ValueError(f"{what}: a page must be contiguous and pages must not overlap")
    return pages, heads, ps, hd, k0, v0


@functools.lru_cache(maxsize=16)
def _turns(theta: float, half: int):
    return (ctypes.c_double * half)(*[theta ** (-j / half) / (2 * math.pi) for j in range(half)])


def append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, theta: float) -> torch.Tensor:
    """New tokens' packed rows [tokens, (q_heads + 2 kv_heads) * head_dim] (row stride allowed): returns q [tokens, q_heads * head_dim], rotated by
    each token's own position (pairs j, j + head_dim / 2; theta <= 0: not rotated), and writes rotated k and v to their slots.  A slot that is
    not in the pool (-1) is left out."""
    pages, kvh, ps, hd, k_step, v_step = _pool("append", k_pages.shape, k_pages.stride(), v_pages.shape, v_pages.stride(), k_pages.dtype, v_pages.dtype, qkv.dtype)
    tokens, width = qkv.shape if qkv.dim() == 2 else (-1, 0)
    qh = width // hd - 2 * kvh
    if tokens < 0 or width % hd or qh < 1:
        raise ValueError(f"append: rows of q, k and v heads of {hd} expected, with {kvh} k and v heads")
    if positions.numel() != tokens or slots.numel() != tokens:
        raise ValueError("append: one position and one slot for each row")
    _int32("append", positions, slots)
    _same_device("append", qkv, positions, slots, k_pages, v_pages)
    if not qkv.is_cuda:
        x = qkv.float().reshape(tokens, qh + 2 * kvh, hd)
        if theta > 0:
            a = positions.double()[:, None] * torch.tensor(list(_turns(theta, hd // 2)), dtype=torch.float64) * (2 * math.pi)
            cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
            lo, hi = x[:, :qh + kvh, :hd // 2], x[:, :qh + kvh, hd // 2:]
            x = torch.cat([torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1), x[:, qh + kvh:]], 1)
        x = x.to(qkv.dtype)
        there = (slots >= 0) & (slots < pages * ps)
        at = slots[there].long()
        k_pages[at // ps, :, at % ps] = x[there, qh:qh + kvh]
        v_pages[at // ps, :, at % ps] = x[there, qh + kvh:]
        return x[:, :qh].reshape(tokens, qh * hd)
    qkv, row_stride = _aligned_rows(qkv, tokens, width)
    q = qkv.new_empty_strided((tokens, qh * hd), (qh * hd, 1))
    turns = ctypes.addressof(_turns(float(theta), hd // 2)) if theta > 0 else None
    K._launch(N.require().oa_paged_append(K.dt(qkv), qkv.data_ptr(), row_stride, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                          k_step, v_step, positions.data_ptr(), slots.data_ptr(), turns, tokens, qh, kvh, hd, ps,
                                          pages, N.stream()), "oa_paged_append")
    return q


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor,
              max_fresh: int, prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0, scale: Optional[float] = None,
              return_lse: bool = False):
    """Attention of the new tokens q [tokens, q_heads * head_dim] (row stride allowed) of a batch: token i of the n new ones of a request (rows
    starts[b] .. starts[b + 1], at most `max_fresh`) sees the whole shared prompt, `prefix_len` keys in the pages of `prefix_table`, and the
    first lens[b] - n + i + 1 keys of its own pages.  q_heads is a multiple of kv_heads.  Returns [tokens, q_heads * head_dim] and, with
    return_lse, also the natural log-sum-exp [tokens, q_heads] fp32.  Rows that see nothing, and rows of no request, are 0 (-inf).

    bf16 with heads of 64 or 128, up to 2048 requests, runs on the tensor cores: weights are rounded to bf16 before they meet the values, sums are
    fp32, and a value of a request's new tokens that is not finite may reach its earlier new tokens too.  All else takes a block to a row."""
    batch = lens.numel()
    (pages, kvh, ps, hd, k_step, v_step, tokens, cols, qh, width, table_stride, scale, need) = _attention_layout(
        q.shape, q.dtype, k_pages.shape, k_pages.stride(), v_pages.shape, v_pages.stride(), k_pages.dtype, v_pages.dtype, tables.shape, tables.stride(),
        tables.dtype, batch, starts.numel(), max_fresh, None if prefix_table is None else prefix_table.numel(), prefix_len, scale, q.get_device())
    if prefix_len > 0:
        _int32("attention", lens, starts, prefix_table)
        _same_device("attention", q, k_pages, v_pages, tables, lens, starts, prefix_table)
    else:
        _int32("attention", lens, starts)
        _same_device("attention", q, k_pages, v_pages, tables, lens, starts)
    if not q.is_cuda:
        return _attention_cpu(q, k_pages, v_pages, tables, lens, starts, max_fresh, prefix_table, prefix_len, scale, return_lse)
    q, q_step = _aligned_rows(q, tokens, cols)
    out = q.new_empty_strided((tokens, cols), (cols, 1))
    lse = torch.empty_strided((tokens, qh), (qh, 1), dtype=torch.float32, device=q.device) if return_lse else None
    code = K.dt(q)
    # scratch of the call's own: calls on several streams do not meet in it
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    K._launch(N.require().oa_paged_attn(code, q.data_ptr(), q_step, k_pages.data_ptr(), v_pages.data_ptr(), k_step, v_step, tables.data_ptr(), table_stride,
                                        lens.data_ptr(), starts.data_ptr(), N.ptr(prefix_table), prefix_len, out.data_ptr(), N.ptr(lse), tokens, batch,
                                        max_fresh, qh, kvh, hd, ps, pages, width, scale, N.ptr(scratch), K.status_word(q.device).data_ptr(), N.stream()),
              "oa_paged_attn", 2 if need else 1, outputs=(out,))
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def _attention_layout(q_shape, dtype, k_shape, k_stride, v_shape, v_stride, k_dtype, v_dtype, t_shape, t_stride, t_dtype, batch, n_starts, max_fresh, n_prefix,
                      prefix_len, scale, device):
    """The checks of `attention`; (.. of the pool, tokens, columns, query heads, table width and row stride, scale, bytes of scratch on
    the device, -1 being the CPU)."""
    pool = _pool("attention", k_shape, k_stride, v_shape, v_stride, k_dtype, v_dtype, dtype)
    pages, kvh, ps, hd = pool[:4]
    tokens, cols = q_shape if len(q_shape) == 2 else (0, 0)
    if cols == 0 or cols % (hd * kvh):
        raise ValueError(f"attention: q must be [tokens, q_heads * {hd}] with q_heads a multiple of {kvh}")
    if n_starts != batch + 1 or max_fresh < 0 or prefix_len < 0:
        raise ValueError("attention: starts has one entry more than lens; max_fresh and prefix_len are not negative")
    if prefix_len > 0 and (n_prefix is None or n_prefix * ps < prefix_len):
        raise ValueError(f"attention: prefix_table holds fewer than {prefix_len} tokens")
    width, table_stride = _table_layout("attention", t_shape, t_stride, t_dtype, batch)
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    qh = cols // hd
    code = K._DT.get(dtype) if device >= 0 else None
    need = N.require().oa_paged_attn_scratch_bytes(code, tokens, batch, max_fresh, qh, kvh, hd, pages, prefix_len, scale) if code is not None else 0
    return (*pool, tokens, cols, qh, width, table_stride, scale, need)


def _attention_cpu(q, k_pages, v_pages, tables, lens, starts, max_fresh, prefix_table, prefix_len, scale, return_lse):
    pages, kvh, ps, hd = k_pages.shape
    tokens, qh = q.shape[0], q.shape[1] // hd
    out = torch.zeros((tokens, qh, hd))
    lse = torch.full((tokens, qh), -math.inf)

    def keys(pool, table, n):
        at = torch.arange(n)
        page = table.long()[at // ps] if n else at
        live = (page >= 0) & (page < pages)
        x = pool[page.clamp(0, max(pages - 1, 0)), :, at % ps].float() * live[:, None, None]
        return x.repeat_interleave(qh // kvh, 1)

    for b in range(lens.numel()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        own = min(int(lens[b]), tables.shape[1] * ps)
        for i in range(min(hi - lo, max_fresh, tokens - lo)):
            n = max(own - (hi - lo) + i + 1, 0)
            if n + prefix_len == 0:
                continue
            k, v = (torch.cat([keys(p, prefix_table, prefix_len), keys(p, tables[b], n)] if prefix_len else [keys(p, tables[b], n)]) for p in (k_pages, v_pages))
            x = torch.einsum("hd,shd->hs", q[lo + i].float().reshape(qh, hd), k) * scale
            lse[lo + i] = torch.logsumexp(x, -1)
            out[lo + i] = torch.einsum("hs,shd->hd", torch.softmax(x, -1), v)
    out = out.reshape(tokens, qh * hd).to(q.dtype)
    return (out, lse) if return_lse else out
