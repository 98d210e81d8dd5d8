"""Log-probabilities of given tokens, with the entropy of every row and its likeliest tokens, and the logits' gradient, on raw tensors.

What scores a prompt, reports a drawn token beside its alternatives, and trains a policy.  CUDA tensors run csrc/kernels/logprob.cu, whose head
states the mathematics; CPU tensors the plain statement of it.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional

import torch

from .. import _native as N
from . import kernels as K
from .packed import _copied, _overlap, _step, _stream, _together, _whole

MAX_TOP = 32


class TokenLogProbs(NamedTuple):
    logprobs: torch.Tensor          # [rows] fp32, of the targets
    entropy: torch.Tensor           # [rows] fp32, natural units
    stats: torch.Tensor             # [rows, 2] fp32: a row's largest scaled logit, and the logarithm of its sum of exponentials less that
    top_logprobs: torch.Tensor      # [rows, top] fp32
    top_ids: torch.Tensor           # [rows, top] int32, the likeliest first


@functools.lru_cache(maxsize=256)
def _layout(what, shape, stride, dtype, t_shape, t_stride, t_dtype, scale, top, ignore_index):
    """The checks that shapes and types allow; elements between the rows of logits, None where they are copied."""
    if len(shape) != 2 or dtype not in (torch.float32, torch.bfloat16) or not 1 <= shape[1] < 1 << 30 or shape[0] >= 1 << 30:
        raise ValueError(f"{what}: logits must be float32 or bfloat16 [rows, vocab]")
    rows, vocab = shape
    if t_dtype is not torch.int32 or t_shape != (rows,) or (rows > 1 and t_stride != (1,)):
        raise ValueError(f"{what}: targets must be a contiguous int32 tensor [{rows}]")
    if not 0 < scale < math.inf:
        raise ValueError(f"{what}: scale must be positive, not {scale}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"{what}: 0 to {min(MAX_TOP, vocab)} alternatives, not {top}")
    if not -2 ** 31 <= ignore_index < 2 ** 31:
        raise ValueError(f"{what}: ignore_index is one of the targets' 32 bits, not {ignore_index}")
    return None if stride[1] != 1 and vocab > 1 else vocab if rows <= 1 else stride[0]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, scale: float = 1.0, ignore_index: int = -100) -> TokenLogProbs:
    """Of every row of scale * logits [rows, vocab] (row stride allowed; scale is 1 / temperature): the log-probability of its target, the entropy, and
    the `top` likeliest tokens (at most 32) with theirs; equal logits rank by index.  A target of ignore_index has log-probability 0, any other that is
    no token NaN.  Logits of -inf have probability 0; a row with NaN or +inf is NaN; one without anything above -inf has log-probabilities of
    -inf and entropy 0.  The same call gives the same bits; the last bits of a row depend on the order of its sums, which goes by where it begins (from a
    multiple of 16 bytes or not), `top` and the number of rows."""
    scale, top, ignore_index = float(scale), _whole(top), _whole(ignore_index)
    step = _layout("token_logprobs", logits.shape, logits.stride(), logits.dtype, targets.shape, targets.stride(), targets.dtype, scale, top, ignore_index)
    device = _together("token_logprobs", logits, targets)
    if device < 0:
        return _cpu(logits, targets, top, scale, ignore_index)
    rows, vocab = logits.shape
    if step is None:
        logits, step = _copied(logits), vocab
    f32 = torch.empty(rows * (4 + 2 * top), dtype=torch.float32, device=logits.device)
    if top:
        logprobs, entropy, stats, top_logprobs, top_ids = torch.unsafe_split_with_sizes(f32, (rows, rows, 2 * rows, top * rows, top * rows))
        top_logprobs, top_ids = top_logprobs.view(rows, top), top_ids.view(torch.int32).view(rows, top)
    else:
        logprobs, entropy, stats = torch.unsafe_split_with_sizes(f32, (rows, rows, 2 * rows))
        top_logprobs = f32.as_strided((rows, 0), (1, 1))         # without elements: not worth two allocations
        top_ids = top_logprobs.view(torch.int32)
    at = f32.data_ptr()
    K._launch(N.require().oa_token_logprobs(K.dt(logits), logits.data_ptr(), step, targets.data_ptr(), at, at + 4 * rows, at + 8 * rows, at + 16 * rows,
                                            at + 4 * (4 + top) * rows, top, rows, vocab, scale, ignore_index, _stream(device)),
              "oa_token_logprobs", outputs=(logprobs, entropy))
    return TokenLogProbs(logprobs, entropy, stats.view(rows, 2), top_logprobs, top_ids)


@torch.no_grad()
def _cpu(logits, targets, top, scale, ignore_index):
    rows, vocab = logits.shape
    logits = logits.contiguous()
    y = logits.float() * scale
    bad = ~(y <= torch.finfo(torch.float32).max).all(1)
    m = torch.where(bad, math.nan, y.amax(1))
    none = m == -math.inf
    d = torch.where(none[:, None], -math.inf, y - m[:, None])
    log_l = torch.where(none, 0.0, torch.exp(d).sum(1).log())
    logp = d - log_l[:, None]
    p = torch.exp(logp)
    entropy = torch.where(none, 0.0, -torch.where((p > 0) | p.isnan(), p * logp, 0.0).sum(1))
    there = (targets >= 0) & (targets < vocab)
    chosen = logp.gather(1, targets.clamp(0, vocab - 1).long()[:, None])[:, 0]
    chosen = torch.where(targets == ignore_index, 0.0, torch.where(there, chosen, math.nan))
    rank = torch.where(logits.isnan(), -math.inf, logits.float())
    ids = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :top]
    return TokenLogProbs(chosen, entropy, torch.stack([m, log_l], 1), logp.gather(1, ids), ids.to(torch.int32))


def token_logprobs_backward(logits: torch.Tensor, targets: torch.Tensor, result: TokenLogProbs, dlogprobs: Optional[torch.Tensor],
                            dentropy: Optional[torch.Tensor] = None, scale: float = 1.0, ignore_index: int = -100,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits' gradient from those of the log-probabilities and of the entropy ([rows] fp32, or None for none), given what `token_logprobs` returned
    for the same logits, targets, scale and ignore_index.  `out` (row stride allowed) may be the logits themselves.  A row whose target is ignore_index
    takes no part in dlogprobs; one with another target that is no token is NaN; one without anything above -inf is 0."""
    scale, ignore_index = float(scale), _whole(ignore_index)
    step = _layout("token_logprobs_backward", logits.shape, logits.stride(), logits.dtype, targets.shape, targets.stride(), targets.dtype, scale, 0, ignore_index)
    rows, vocab = logits.shape
    for name, t, shape in (("dlogprobs", dlogprobs, (rows,)), ("dentropy", dentropy, (rows,)), ("result.entropy", result.entropy, (rows,)),
                           ("result.stats", result.stats, (rows, 2))):
        if t is not None and (t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous()):
            raise ValueError(f"token_logprobs_backward: {name} must be a contiguous float32 tensor {list(shape)}")
    device = _together("token_logprobs_backward", logits, targets, result.entropy, result.stats, *(t for t in (dlogprobs, dentropy, out) if t is not None))
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        to = vocab
    else:
        to = _step(out.shape, out.stride()) if out.dim() == 2 else None
        if out.shape != logits.shape or out.dtype is not logits.dtype or to is None:
            raise ValueError(f"token_logprobs_backward: out must be {logits.dtype} {list(logits.shape)}, the elements of a row side by side, rows apart")
        if (out.data_ptr() != logits.data_ptr() or out.stride() != logits.stride()) and _overlap(out, logits):
            raise ValueError("token_logprobs_backward: out must be the logits or lie apart from them")
    if device < 0:
        return _backward_cpu(logits, targets, result, dlogprobs, dentropy, scale, ignore_index, out)
    if step is None:
        logits, step = _copied(logits), vocab
    K._launch(N.require().oa_token_logprobs_bwd(K.dt(logits), logits.data_ptr(), step, targets.data_ptr(), result.entropy.data_ptr(),
                                                result.stats.data_ptr(), N.ptr(dlogprobs), N.ptr(dentropy), out.data_ptr(), to, rows, vocab, scale, ignore_index,
                                                _stream(device)), "oa_token_logprobs_bwd", outputs=(out,))
    return out


@torch.no_grad()
def _backward_cpu(logits, targets, result, dlogprobs, dentropy, scale, ignore_index, out):
    rows, vocab = logits.shape
    m, log_l = result.stats[:, :1], result.stats[:, 1:]
    none = m == -math.inf
    there = (targets >= 0) & (targets < vocab)
    g = torch.zeros(rows) if dlogprobs is None else torch.where(targets == ignore_index, 0.0, torch.where(there, dlogprobs, math.nan))
    h = torch.zeros(rows) if dentropy is None else dentropy
    logp = torch.where(none, -math.inf, logits.float() * scale - m) - log_l
    p = torch.exp(logp)
    d = -p * (g[:, None] + h[:, None] * (torch.where((p > 0) | p.isnan(), logp, 0.0) + result.entropy[:, None]))
    d[there.nonzero()[:, 0], targets[there].long()] += g[there]
    out.copy_(torch.where(none, 0.0, scale * d))
    return out
