"""Sequences of different lengths packed one behind the other, on raw tensors: rotary positions with several axes, causal attention with grouped
heads and its gradients.

Layout contract: every tensor has one row to a token; sequence b is rows starts[b] .. starts[b + 1] (int32, on the device).  Heads lie side by side in
a row, query head h reads key-value head h / (q_heads / kv_heads), and q, k and v may be slices of one projection's rows.  `plan` works out once for a
batch what the attention kernels work on; all layers use it, in both directions.  Sequences do not reach one another, whatever they hold; rows of
no sequence (behind the last one, say) are neither read nor reach anything, and are 0 in what comes back.

The form for single tokens over a cache is `paged.append` (theta 0, for rows that `rotary` turned) with `paged.attention`.

CUDA tensors run csrc/kernels/packed.cu, packed_attn.cu, packed_short.cu and packed_attn_f32.cu; CPU tensors the plain statement of the same mathematics.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional, Sequence

import torch

from .. import _native as N
from . import kernels as K

HEAD_DIMS = (64, 128)           # of the bf16 attention kernels; fp32 and the CPU path take any up to 128
MAX_AXES = 8
MAX_PAIRS = 128
_FLOATS = (torch.float32, torch.bfloat16)


class PackedPlan(NamedTuple):
    """What the attention kernels work on, for one batch of packed sequences."""
    starts: torch.Tensor                # [batch + 1] int32, rising and within [0, tokens]
    words: Optional[torch.Tensor]       # the kernels' lists of tiles; None on the CPU
    tokens: int
    batch: int


def _current(what: str, t: torch.Tensor) -> None:
    if t.is_cuda and t.get_device() != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors on {t.device}, but the current device is cuda:{torch.cuda.current_device()}")


def _together(what: str, first: torch.Tensor, *tensors: torch.Tensor) -> None:
    at = first.get_device()
    for t in tensors:
        if t.get_device() != at:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")
    _current(what, first)


def _rows(t: torch.Tensor, aligned: bool):
    """(the rows as the kernels read them, elements between rows): elements side by side and, if `aligned`, every row on 16 bytes.  A copy where they
    are not."""
    rows, cols = t.shape
    step, unit = t.stride()
    if rows <= 1:
        step = cols                                  # the stride of a single row says nothing
        if aligned:
            step += -step % 8
    if (unit == 1 or cols <= 1) and step >= cols and (not aligned or (step * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0)):
        return t, step
    if aligned and cols * t.element_size() % 16:     # rows of whole heads never are
        raise ValueError(f"packed: rows of {cols} elements do not fill 16-byte pieces")
    return (t.clone(memory_format=torch.contiguous_format) if t.is_contiguous() else K.contiguous(t)), cols


def plan(starts: torch.Tensor, tokens: int) -> PackedPlan:
    """What `attention` needs to know about sequences whose rows begin at `starts` [batch + 1] (int32; the last entry is the end of the last one) in
    tensors of `tokens` rows.  Starts that fall, or leave [0, tokens], count as the nearest ones that do not.  Nothing is read back to the host."""
    if starts.dtype is not torch.int32 or starts.dim() != 1 or not starts.is_contiguous() or starts.numel() < 1:
        raise ValueError("plan: starts must be a contiguous int32 tensor [batch + 1]")
    batch = starts.numel() - 1
    if not 0 <= tokens <= 1 << 30 or batch > 1 << 24:
        raise ValueError(f"plan: {batch} sequences in {tokens} rows; at most {1 << 24} in {1 << 30}")
    if not starts.is_cuda:
        return PackedPlan(torch.cummax(starts.clamp(0, tokens), 0).values, None, tokens, batch)
    _current("plan", starts)
    words = torch.empty(N.require().oa_packed_plan_bytes(tokens, batch) // 4, dtype=torch.int32, device=starts.device)
    K._launch(N.require().oa_packed_plan(starts.data_ptr(), words.data_ptr(), batch, tokens, N.stream()), "oa_packed_plan")
    return PackedPlan(words[8:8 + batch + 1], words, tokens, batch)


@functools.lru_cache(maxsize=64)
def _rotary_tables(pair_axes: tuple, theta: float):
    half = len(pair_axes)
    return (ctypes.c_uint8 * half)(*pair_axes), (ctypes.c_double * half)(*[theta ** (-j / half) / (2 * math.pi) for j in range(half)])


def rotary(x: torch.Tensor, positions: torch.Tensor, pair_axes: Sequence[int], heads: int, head_dim: int, theta: float, backward: bool = False,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The first `heads` heads of every row of x [tokens, >= heads * head_dim] (row stride allowed) turned by their token's positions [axes, tokens]
    (int32): pair j of a head, dimensions j and j + len(pair_axes), by theta^(-j / len(pair_axes)) times the position on axis pair_axes[j].  Dimensions from
    2 len(pair_axes) on stay as they are.  One axis and half the head's dimensions make the usual rotary embedding.  `backward`: the other way round,
    which is the gradient.  Returns [tokens, heads * head_dim], `out` if given, which may be x itself or its first columns."""
    pair_axes = tuple(int(a) for a in pair_axes)
    if x.dim() != 2 or heads < 1 or head_dim < 2 or x.shape[1] < heads * head_dim or x.dtype not in _FLOATS:
        raise ValueError(f"rotary: x must be float32 or bfloat16 [tokens, >= {heads} * {head_dim}]")
    tokens, cols = x.shape[0], heads * head_dim
    if not 1 <= len(pair_axes) <= min(head_dim // 2, MAX_PAIRS):
        raise ValueError(f"rotary: 1 to {min(head_dim // 2, MAX_PAIRS)} pairs of a head of {head_dim}, not {len(pair_axes)}")
    if positions.dtype is not torch.int32 or positions.dim() != 2 or not positions.is_contiguous() or positions.shape[1] != tokens \
            or not 1 <= positions.shape[0] <= MAX_AXES:
        raise ValueError(f"rotary: positions must be a contiguous int32 tensor [axes, {tokens}] of at most {MAX_AXES} axes")
    if min(pair_axes) < 0 or max(pair_axes) >= positions.shape[0]:
        raise ValueError(f"rotary: pair_axes names axes that positions [{positions.shape[0]}, tokens] do not have")
    if not 0 < theta < math.inf:
        raise ValueError(f"rotary: theta must be positive, not {theta}")
    _together("rotary", x, positions)
    if out is None:
        out = x.new_empty((tokens, cols))
    else:
        if out.dim() != 2 or out.shape[0] != tokens or out.shape[1] < cols or out.dtype is not x.dtype:
            raise ValueError(f"rotary: out must be {x.dtype} [{tokens}, >= {cols}]")
        if (out.shape[1] > 1 and out.stride(1) != 1) or (tokens > 1 and out.stride(0) < cols):
            raise ValueError("rotary: out must have the elements of a row side by side and rows that do not overlap")
        _together("rotary", x, out)
        out = out[:, :cols]
    axes, turns = _rotary_tables(pair_axes, float(theta))
    if not x.is_cuda:
        half = len(pair_axes)
        a = positions.double()[list(pair_axes)].t() * torch.tensor(list(turns), dtype=torch.float64) * (2 * math.pi)
        cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
        sin = -sin if backward else sin
        v = x[:, :cols].float().reshape(tokens, heads, head_dim)
        lo, hi = v[..., :half], v[..., half:2 * half]
        out.copy_(torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, v[..., 2 * half:]], -1).reshape(tokens, cols))
        return out
    x = x[:, :cols]
    x, step = _rows(x, False)
    K._launch(N.require().oa_rotary_axes(K.dt(x), x.data_ptr(), step, out.data_ptr(), out.stride(0) if tokens > 1 else cols, positions.data_ptr(),
                                         ctypes.addressof(axes), ctypes.addressof(turns), len(pair_axes), tokens, heads, head_dim, int(backward),
                                         N.stream()), "oa_rotary_axes", outputs=(out,))
    return out


def _heads(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan, head_dim: int):
    """The checks of both directions: (query heads, key-value heads)."""
    if q.dtype not in _FLOATS or k.dtype is not q.dtype or v.dtype is not q.dtype or q.dim() != 2 or k.dim() != 2 or v.shape != k.shape:
        raise ValueError(f"{what}: q, k and v must be float32 or bfloat16 matrices of one type, k and v of one shape")
    if head_dim < 1 or q.shape[1] < 1 or k.shape[1] < 1 or k.shape[1] % head_dim or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: rows of heads of {head_dim}, the query heads a multiple of the key-value heads; not {q.shape[1]} and {k.shape[1]} columns")
    if q.shape[0] != plan.tokens or k.shape[0] != plan.tokens:
        raise ValueError(f"{what}: the plan is for {plan.tokens} rows, not {q.shape[0]} and {k.shape[0]}")
    _together(what, q, k, v, plan.starts)
    if q.is_cuda:
        if q.dtype is torch.bfloat16 and head_dim not in HEAD_DIMS:
            raise ValueError(f"{what}: bfloat16 heads of one of {HEAD_DIMS}, not of {head_dim}")
        if head_dim > 128:
            raise ValueError(f"{what}: heads of at most 128, not of {head_dim}")
    return q.shape[1] // head_dim, k.shape[1] // head_dim


def _scale(what: str, scale: Optional[float], head_dim: int) -> float:
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"{what}: scale must be positive, not {scale}")
    return scale


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan, head_dim: int, scale: Optional[float] = None, return_lse: bool = False):
    """Causal attention within every sequence: q [tokens, q_heads * head_dim], k and v [tokens, kv_heads * head_dim] (row strides allowed), q_heads a
    multiple of kv_heads.  Returns [tokens, q_heads * head_dim] and, with return_lse, also the natural log-sum-exp [q_heads, tokens] fp32, which the
    gradients need.  `scale` defaults to head_dim^-1/2.  Rows of no sequence are 0 (-inf).

    bf16 (heads of 64 or 128) runs on the tensor cores: weights are rounded to bf16 before they meet the values, sums are fp32.  A value that is not finite
    may reach earlier tokens of its own sequence, as its weight there is 0 times it."""
    hq, hk = _heads("attention", q, k, v, plan, head_dim)
    scale = _scale("attention", scale, head_dim)
    if not q.is_cuda:
        o, lse = _attention_cpu(q, k, v, plan, head_dim, scale)
        return (o.to(q.dtype), lse) if return_lse else o.to(q.dtype)
    half = q.dtype is torch.bfloat16
    (q, qs), (k, ks), (v, vs) = (_rows(t, half) for t in (q, k, v))
    o = q.new_empty((plan.tokens, hq * head_dim))
    lse = torch.empty((hq, plan.tokens), dtype=torch.float32, device=q.device) if return_lse else None
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), plan.words.data_ptr(), o.data_ptr(), N.ptr(lse), plan.tokens, plan.batch, hq, hk, head_dim, qs, ks, vs,
            hq * head_dim, scale)
    if half:
        K._launch(N.require().oa_packed_attn(*args, K.status_word(q.device).data_ptr(), N.stream()), "oa_packed_attn", 2, outputs=(o,))
    else:
        K._launch(N.require().oa_packed_attn_f32(*args, N.stream()), "oa_packed_attn_f32", outputs=(o,))
    return (o, lse) if return_lse else o


def _attention_cpu(q, k, v, plan, head_dim, scale):
    """(o, lse) in fp32, differentiable."""
    hq, hk = q.shape[1] // head_dim, k.shape[1] // head_dim
    out = torch.zeros((plan.tokens, hq * head_dim))
    lse = torch.full((hq, plan.tokens), -math.inf)
    parts, starts = [], plan.starts.tolist()
    for lo, hi in zip(starts, starts[1:]):
        if hi > lo:
            qs, ks, vs = (t[lo:hi].float().reshape(hi - lo, -1, head_dim) for t in (q, k, v))
            ks, vs = (t.repeat_interleave(hq // hk, 1) for t in (ks, vs))
            x = torch.einsum("ihd,jhd->hij", qs, ks) * scale
            x = x.masked_fill(torch.ones(hi - lo, hi - lo, dtype=torch.bool).triu(1), -math.inf)
            lse[:, lo:hi] = torch.logsumexp(x.detach(), -1)
            parts.append((lo, hi, torch.einsum("hij,jhd->ihd", torch.softmax(x, -1), vs).reshape(hi - lo, -1)))
    for lo, hi, y in parts:
        out[lo:hi] = y
    return out, lse


def attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, dout: torch.Tensor, lse: torch.Tensor, plan: PackedPlan,
                       head_dim: int, scale: Optional[float] = None, dqkv: Optional[torch.Tensor] = None):
    """The gradients (dq, dk, dv) of `attention` from its inputs, its output and log-sum-exp, and dout [tokens, q_heads * head_dim] (row stride
    allowed).  They are slices of `dqkv` [tokens, (q_heads + 2 kv_heads) * head_dim], a packed projection's gradient.  Those of a key-value head are the
    sums over the query heads that share it, added up in one order: the same inputs give the same bits.  Rows of no sequence are 0."""
    hq, hk = _heads("attention_backward", q, k, v, plan, head_dim)
    scale = _scale("attention_backward", scale, head_dim)
    if o.shape != q.shape or dout.shape != q.shape or o.dtype is not q.dtype or dout.dtype is not q.dtype:
        raise ValueError(f"attention_backward: o and dout must be {q.dtype} {list(q.shape)}")
    if lse.shape != (hq, plan.tokens) or lse.dtype is not torch.float32 or not lse.is_contiguous():
        raise ValueError(f"attention_backward: lse must be a contiguous float32 tensor [{hq}, {plan.tokens}]")
    cols = [hq * head_dim, hk * head_dim, hk * head_dim]
    if dqkv is None:
        dqkv = q.new_empty((plan.tokens, sum(cols)))
    elif dqkv.shape != (plan.tokens, sum(cols)) or dqkv.dtype is not q.dtype or not dqkv.is_contiguous():
        raise ValueError(f"attention_backward: dqkv must be a contiguous {q.dtype} tensor [{plan.tokens}, {sum(cols)}]")
    _together("attention_backward", q, o, dout, lse, dqkv)
    grads = torch.split(dqkv, cols, 1)
    if not q.is_cuda:
        with torch.enable_grad():
            leaves = [t.detach().float().requires_grad_(True) for t in (q, k, v)]
            y, _ = _attention_cpu(*leaves, plan, head_dim, scale)
            got = torch.autograd.grad(y, leaves, dout.float(), allow_unused=True) if y.requires_grad else (None,) * 3
        for to, g in zip(grads, got):
            to.copy_(g) if g is not None else to.zero_()
        return grads
    half = q.dtype is torch.bfloat16
    (q, qs), (k, ks), (v, vs), (o, os), (dout, dos) = (_rows(t, half) for t in (q, k, v, o, dout))
    dq, dk, dv = grads
    if half and dqkv.data_ptr() % 16:
        raise ValueError("attention_backward: dqkv must begin on 16 bytes")
    width = dqkv.shape[1]
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(), lse.data_ptr(), plan.words.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), plan.tokens, plan.batch, hq, hk, head_dim, qs, ks, vs, os, dos, width, width, width, scale)
    if half:
        # scratch of the call's own: calls on several streams, and graphs, do not meet in it
        need = N.require().oa_packed_attn_bwd_scratch_bytes(plan.tokens, plan.batch, hq, hk, head_dim)
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
        K._launch(N.require().oa_packed_attn_bwd(*args, scratch.data_ptr(), K.status_word(q.device).data_ptr(), N.stream()), "oa_packed_attn_bwd", 4,
                  outputs=(dqkv,))
    else:
        K._launch(N.require().oa_packed_attn_f32_bwd(*args, N.stream()), "oa_packed_attn_f32_bwd", outputs=(dqkv,))
    return grads
