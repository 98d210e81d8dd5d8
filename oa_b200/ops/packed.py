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
import operator
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


def _together(what: str, first: torch.Tensor, *tensors: torch.Tensor) -> int:
    """The device that all tensors are on (-1: the CPU); a CUDA one has to be the current one, whose stream the kernels go to."""
    at = first.get_device()
    for t in tensors:
        if t.get_device() != at:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")
    if at >= 0 and at != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors on {first.device}, but the current device is cuda:{torch.cuda.current_device()}")
    return at


def _whole(x) -> int:
    """What the checks below are remembered by has to be plain numbers: a tensor is the same key whatever it holds by now."""
    return x if type(x) is int else operator.index(x)


def _stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _step(shape, stride) -> Optional[int]:
    """Elements between the rows of a matrix whose rows have their elements side by side and do not overlap; None otherwise."""
    rows, cols = shape
    if cols > 1 and stride[1] != 1:
        return None
    return cols if rows <= 1 else stride[0] if stride[0] >= cols else None      # the stride of a single row says nothing


def _copied(t: torch.Tensor) -> torch.Tensor:
    return t.clone(memory_format=torch.contiguous_format) if t.is_contiguous() else K.contiguous(t)


def _end(t: torch.Tensor) -> int:
    """The address behind a matrix's last element."""
    (rows, cols), (down, right) = t.shape, t.stride()
    return t.data_ptr() + ((rows - 1) * down + (cols - 1) * right + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices share memory (columns of one buffer that lie beside one another do not)."""
    if not a.numel() or not b.numel():
        return False
    lo, lo2 = a.data_ptr(), b.data_ptr()
    if (lo2 >= _end(a)) if lo <= lo2 else (lo >= _end(b)):
        return False
    pitch = a.stride(0) * a.element_size()
    if a.stride(1) == b.stride(1) == 1 and b.stride(0) * b.element_size() == pitch > 0:
        at = (lo2 - lo) % pitch
        return at < a.shape[1] * a.element_size() or at + b.shape[1] * b.element_size() > pitch
    return True


def _apart(what: str, out: torch.Tensor, *tensors: torch.Tensor) -> None:
    if not out.numel():
        return
    lo, hi = out.data_ptr(), _end(out)
    for t in tensors:
        at = t.data_ptr()
        if at < hi and (at >= lo or _end(t) > lo) and _overlap(out, t):
            raise ValueError(f"{what}: the result's memory is that of an operand")


def plan(starts: torch.Tensor, tokens: int) -> PackedPlan:
    """What `attention` needs to know about sequences whose rows begin at `starts` [batch + 1] (int32; the last entry is the end of the last one) in
    tensors of `tokens` rows.  Starts that fall, or leave [0, tokens], count as the nearest ones that do not.  Nothing is read back to the host."""
    tokens = _whole(tokens)
    if starts.dtype is not torch.int32 or starts.dim() != 1 or not starts.is_contiguous() or starts.numel() < 1:
        raise ValueError("plan: starts must be a contiguous int32 tensor [batch + 1]")
    batch = starts.numel() - 1
    if not 0 <= tokens <= 1 << 30 or batch > 1 << 24:
        raise ValueError(f"plan: {batch} sequences in {tokens} rows; at most {1 << 24} in {1 << 30}")
    if not starts.is_cuda:
        return PackedPlan(torch.cummax(starts.clamp(0, tokens), 0).values, None, tokens, batch)
    device = _together("plan", starts)
    words = torch.empty(N.require().oa_packed_plan_bytes(tokens, batch) // 4, dtype=torch.int32, device=starts.device)
    K._launch(N.require().oa_packed_plan(starts.data_ptr(), words.data_ptr(), batch, tokens, _stream(device)), "oa_packed_plan")
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
    which is the gradient.  Returns [tokens, heads * head_dim], the first columns of `out` if given, which may be x itself but not overlap it otherwise."""
    if type(pair_axes) is not tuple:
        pair_axes = tuple(map(operator.index, pair_axes))
    heads, head_dim, theta = _whole(heads), _whole(head_dim), float(theta)
    step, axes, turns = _rotary_layout(x.shape, x.stride(), x.dtype, positions.shape, positions.stride(), positions.dtype, pair_axes, heads, head_dim, theta)
    tokens, cols = x.shape[0], heads * head_dim
    if out is None:
        device = _together("rotary", x, positions)
        out, to = x.new_empty((tokens, cols)), cols
    else:
        device = _together("rotary", x, positions, out)
        if out.dim() != 2 or out.shape[0] != tokens or out.shape[1] < cols or out.dtype is not x.dtype:
            raise ValueError(f"rotary: out must be {x.dtype} [{tokens}, >= {cols}]")
        out = out[:, :cols]
        to = _step(out.shape, out.stride())
        if to is None:
            raise ValueError("rotary: out must have the elements of a row side by side and rows that do not overlap")
        if x.data_ptr() != out.data_ptr() or (tokens > 1 and x.stride() != out.stride()):
            _apart("rotary", out, x[:, :cols])
    if device < 0:
        _rotary_cpu(x[:, :cols].reshape(tokens, heads, head_dim), positions, pair_axes, turns, backward, out)
        return out
    if step is None:
        x = _copied(x[:, :cols])
        step = cols
    K._launch(N.require().oa_rotary_axes(K.dt(x), x.data_ptr(), step, out.data_ptr(), to, positions.data_ptr(), ctypes.addressof(axes), ctypes.addressof(turns),
                                         len(pair_axes), tokens, heads, head_dim, int(backward), _stream(device)), "oa_rotary_axes", outputs=(out,))
    return out


@torch.no_grad()
def _rotary_cpu(x, positions, pair_axes, turns, backward, out):
    half = len(pair_axes)
    a = positions.double()[list(pair_axes)].t() * torch.tensor(list(turns), dtype=torch.float64) * (2 * math.pi)
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    sin = -sin if backward else sin
    v = x.float()
    lo, hi = v[..., :half], v[..., half:2 * half]
    out.copy_(torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, v[..., 2 * half:]], -1).reshape(out.shape))


# What follows from shapes, strides and types alone is worked out once for each of them: the checks took longer than a small launch.
@functools.lru_cache(maxsize=256)
def _rotary_layout(shape, stride, dtype, p_shape, p_stride, p_dtype, pair_axes, heads, head_dim, theta):
    """The checks of `rotary`; (elements between the rows of x or None where they are copied, the axes and turns of the pairs)."""
    if len(shape) != 2 or heads < 1 or head_dim < 2 or shape[1] < heads * head_dim or dtype not in _FLOATS:
        raise ValueError(f"rotary: x must be float32 or bfloat16 [tokens, >= {heads} * {head_dim}]")
    if not 1 <= len(pair_axes) <= min(head_dim // 2, MAX_PAIRS):
        raise ValueError(f"rotary: 1 to {min(head_dim // 2, MAX_PAIRS)} pairs of a head of {head_dim}, not {len(pair_axes)}")
    if p_dtype is not torch.int32 or len(p_shape) != 2 or p_shape[1] != shape[0] or not 1 <= p_shape[0] <= MAX_AXES \
            or (p_shape[1] > 1 and p_stride[1] != 1) or (p_shape[0] > 1 and 0 < p_shape[1] != p_stride[0]):
        raise ValueError(f"rotary: positions must be a contiguous int32 tensor [axes, {shape[0]}] of at most {MAX_AXES} axes")
    if any(isinstance(a, torch.Tensor) for a in pair_axes):
        raise ValueError("rotary: pair_axes must be whole numbers, not tensors")
    if not all(0 <= operator.index(a) < p_shape[0] for a in pair_axes):
        raise ValueError(f"rotary: pair_axes names axes that positions [{p_shape[0]}, tokens] do not have")
    if not 0 < theta < math.inf:
        raise ValueError(f"rotary: theta must be positive, not {theta}")
    if shape[0] > 1 << 30 or heads * head_dim > 1 << 30:
        raise ValueError(f"rotary: {list(shape)} is too large")
    step = shape[1] if shape[0] <= 1 else stride[0]
    return (step if stride[1] == 1 else None, *_rotary_tables(pair_axes, theta))


@functools.lru_cache(maxsize=256)
def _layout(what, q_shape, q_stride, k_shape, k_stride, v_shape, v_stride, q_dtype, k_dtype, v_dtype, tokens, head_dim, scale, cuda):
    """The checks of both directions; (query heads, key-value heads, scale, elements between the rows of q, of k, of v, or None where they are copied)."""
    if q_dtype not in _FLOATS or k_dtype is not q_dtype or v_dtype is not q_dtype or len(q_shape) != 2 or len(k_shape) != 2 or v_shape != k_shape:
        raise ValueError(f"{what}: q, k and v must be float32 or bfloat16 matrices of one type, k and v of one shape")
    if head_dim < 1 or q_shape[1] < 1 or k_shape[1] < 1 or k_shape[1] % head_dim or q_shape[1] % k_shape[1]:
        raise ValueError(f"{what}: rows of heads of {head_dim}, the query heads a multiple of the key-value heads; not {q_shape[1]} and {k_shape[1]} columns")
    if q_shape[0] != tokens or k_shape[0] != tokens:
        raise ValueError(f"{what}: the plan is for {tokens} rows, not {q_shape[0]} and {k_shape[0]}")
    half = q_dtype is torch.bfloat16
    if cuda:
        if half and head_dim not in HEAD_DIMS:
            raise ValueError(f"{what}: bfloat16 heads of one of {HEAD_DIMS}, not of {head_dim}")
        if head_dim > 128:
            raise ValueError(f"{what}: heads of at most 128, not of {head_dim}")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    if not 0 < scale < math.inf:
        raise ValueError(f"{what}: scale must be positive, not {scale}")
    steps = [_kernel_step(*m, half) for m in ((q_shape, q_stride), (k_shape, k_stride), (v_shape, v_stride))]
    return (q_shape[1] // head_dim, k_shape[1] // head_dim, scale, *steps)


@functools.lru_cache(maxsize=256)
def _backward_layout(forward, o_shape, o_stride, o_dtype, d_shape, d_stride, d_dtype, lse_shape, lse_dtype, lse_side_by_side, batch, device):
    """The checks of the gradients; (query heads, key-value heads, scale, elements between the rows of q, k, v, o and dout or None, columns of dq, dk and
    dv, their sum, bytes of scratch)."""
    q_shape, q_dtype, tokens, head_dim = forward[0], forward[6], forward[9], forward[10]
    hq, hk, scale, *steps = _layout("attention_backward", *forward)
    if o_shape != q_shape or d_shape != q_shape or o_dtype is not q_dtype or d_dtype is not q_dtype:
        raise ValueError(f"attention_backward: o and dout must be {q_dtype} {list(q_shape)}")
    if lse_shape != (hq, tokens) or lse_dtype is not torch.float32 or not lse_side_by_side:
        raise ValueError(f"attention_backward: lse must be a contiguous float32 tensor [{hq}, {tokens}]")
    half = q_dtype is torch.bfloat16
    steps += [_kernel_step(o_shape, o_stride, half), _kernel_step(d_shape, d_stride, half)]
    cols = [hq * head_dim, hk * head_dim, hk * head_dim]
    need = N.require().oa_packed_attn_bwd_scratch_bytes(tokens, batch, hq, hk, head_dim) if half and device >= 0 else 0
    return hq, hk, scale, steps, cols, sum(cols), need


def _kernel_step(shape, stride, half: bool) -> Optional[int]:
    """As _step; the bf16 kernels also want rows 16 bytes apart."""
    step = _step(shape, stride)
    return None if step is not None and half and step % 8 else step


def _operands(half: bool, *pairs):
    """[tensor, elements between rows] of each (tensor, step), copied where the kernels cannot read it as it lies."""
    return [(t, s) if s is not None and not (half and t.data_ptr() & 15) else (_copied(t), t.shape[1]) for t, s in pairs]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan, head_dim: int, scale: Optional[float] = None, return_lse: bool = False):
    """Causal attention within every sequence: q [tokens, q_heads * head_dim], k and v [tokens, kv_heads * head_dim] (row strides allowed), q_heads a
    multiple of kv_heads.  Returns [tokens, q_heads * head_dim] and, with return_lse, also the natural log-sum-exp [q_heads, tokens] fp32, which the
    gradients need.  `scale` defaults to head_dim^-1/2.  Rows of no sequence are 0 (-inf).

    bf16 (heads of 64 or 128) runs on the tensor cores: weights are rounded to bf16 before they meet the values, sums are fp32.  A query or key that is not finite
    reaches no earlier token.  A value (a row of v) that is not finite may reach earlier tokens of its own sequence, in every type and on the CPU: its weight
    there is 0, and 0 times it is NaN."""
    device = _together("attention", q, k, v, plan.starts)
    head_dim, scale = _whole(head_dim), None if scale is None else float(scale)
    hq, hk, scale, *steps = _layout("attention", q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), q.dtype, k.dtype, v.dtype, plan.tokens, head_dim,
                                    scale, device >= 0)
    if device < 0:
        with torch.no_grad():
            o, lse = _attention_cpu(q, k, v, plan, head_dim, scale)
        return (o.to(q.dtype), lse) if return_lse else o.to(q.dtype)
    half = q.dtype is torch.bfloat16
    (q, qs), (k, ks), (v, vs) = _operands(half, (q, steps[0]), (k, steps[1]), (v, steps[2]))
    cols = hq * head_dim
    o = q.new_empty((plan.tokens, cols))
    lse = torch.empty((hq, plan.tokens), dtype=torch.float32, device=q.device) if return_lse else None
    if half:
        K._launch(N.require().oa_packed_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), plan.words.data_ptr(), o.data_ptr(), N.ptr(lse), plan.tokens, plan.batch, hq, hk,
                                             head_dim, qs, ks, vs, cols, scale, K.status_word(q.device).data_ptr(), _stream(device)),
                  "oa_packed_attn", 2, outputs=(o,))
    else:
        K._launch(N.require().oa_packed_attn_f32(q.data_ptr(), k.data_ptr(), v.data_ptr(), plan.words.data_ptr(), o.data_ptr(), N.ptr(lse), plan.tokens, plan.batch, hq,
                                                 hk, head_dim, qs, ks, vs, cols, scale, _stream(device)), "oa_packed_attn_f32", outputs=(o,))
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
    sums over the query heads that share it, added up in one order: the same call gives the same bits, while the order goes by the number of rows and of sequences.  Rows of no sequence are 0.

    bf16: dv takes the weights rounded to bf16.  The score gradients dS go to dq's product as two bf16 numbers and to dk's rounded to one; in sequences of up to 32
    rows to both as two, of 33 to 64 to both as one.  Delta, the row's sum of weights times dP that is taken off in dS, is summed in 32 bits, but for dq of a sequence's
    129th row and on, where it comes from o and dout as they are.  What is not finite may reach the gradients of every token of its sequence."""
    device = _together("attention_backward", q, k, v, o, dout, lse, plan.starts)
    head_dim, scale = _whole(head_dim), None if scale is None else float(scale)
    hq, hk, scale, steps, cols, width, need = _backward_layout(
        (q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), q.dtype, k.dtype, v.dtype, plan.tokens, head_dim, scale, device >= 0),
        o.shape, o.stride(), o.dtype, dout.shape, dout.stride(), dout.dtype, lse.shape, lse.dtype, lse.is_contiguous(), plan.batch, device)
    if dqkv is None:
        dqkv = q.new_empty((plan.tokens, width))
    else:
        if dqkv.shape != (plan.tokens, width) or dqkv.dtype is not q.dtype or not dqkv.is_contiguous():
            raise ValueError(f"attention_backward: dqkv must be a contiguous {q.dtype} tensor [{plan.tokens}, {width}]")
        _together("attention_backward", q, dqkv)
        _apart("attention_backward", dqkv, q, k, v, o, dout, lse)
        if device >= 0 and dqkv.data_ptr() & 15:
            raise ValueError("attention_backward: dqkv must begin on 16 bytes")
    grads = torch.unsafe_split_with_sizes(dqkv, cols, 1)
    if device < 0:
        with torch.inference_mode(False), torch.enable_grad():        # inference mode records nothing, and its tensors cannot be recorded: copies
            leaves = [t.detach().to(torch.float32, copy=True).requires_grad_(True) for t in (q, k, v)]
            y, _ = _attention_cpu(*leaves, plan, head_dim, scale)
            got = torch.autograd.grad(y, leaves, dout.float(), allow_unused=True) if y.requires_grad else (None,) * 3
        for to, g in zip(grads, got):
            to.copy_(g) if g is not None else to.zero_()
        return grads
    half = q.dtype is torch.bfloat16
    (q, qs), (k, ks), (v, vs), (o, os), (dout, dos) = _operands(half, (q, steps[0]), (k, steps[1]), (v, steps[2]), (o, steps[3]), (dout, steps[4]))
    at = dqkv.data_ptr()
    size = dqkv.element_size()
    dk, dv = at + cols[0] * size, at + (cols[0] + cols[1]) * size
    if half:
        # scratch of the call's own: calls on several streams, and graphs, do not meet in it
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
        K._launch(N.require().oa_packed_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(), lse.data_ptr(), plan.words.data_ptr(), at, dk, dv,
                                                 plan.tokens, plan.batch, hq, hk, head_dim, qs, ks, vs, os, dos, width, width, width, scale, scratch.data_ptr(),
                                                 K.status_word(q.device).data_ptr(), _stream(device)), "oa_packed_attn_bwd",
                  5 if need > 8 * hq * plan.tokens + 12 else 4, outputs=(dqkv,))      # a fifth where partial sums are joined
    else:
        K._launch(N.require().oa_packed_attn_f32_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(), lse.data_ptr(), plan.words.data_ptr(), at, dk, dv,
                                                     plan.tokens, plan.batch, hq, hk, head_dim, qs, ks, vs, os, dos, width, width, width, scale, _stream(device)),
                  "oa_packed_attn_f32_bwd", outputs=(dqkv,))
    return grads
