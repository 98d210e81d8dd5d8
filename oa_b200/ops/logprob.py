"""Log-probabilities of given tokens, with the entropy of every row and its likeliest tokens, and the logits' gradient, on raw tensors.

What scores a prompt, reports a drawn token beside its alternatives, and trains a policy.  CUDA tensors run csrc/kernels/logprob.cu, whose head
states the mathematics; CPU tensors the plain statement of it.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from .. import _native as N
from . import kernels as K
from .packed import _together

MAX_TOP = 32


class TokenLogProbs(NamedTuple):
    logprobs: torch.Tensor          # [rows] fp32, of the targets
    entropy: torch.Tensor           # [rows] fp32, natural units
    stats: torch.Tensor             # [rows, 2] fp32: a row's largest scaled logit, and the logarithm of its sum of exponentials less that
    top_logprobs: torch.Tensor      # [rows, top] fp32
    top_ids: torch.Tensor           # [rows, top] int32, the likeliest first


def _check(what: str, logits: torch.Tensor, targets: torch.Tensor, scale: float) -> None:
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or not 1 <= logits.shape[1] < 1 << 31 or logits.shape[0] >= 1 << 31:
        raise ValueError(f"{what}: logits must be float32 or bfloat16 [rows, vocab]")
    if targets.dtype is not torch.int32 or targets.shape != logits.shape[:1] or not targets.is_contiguous():
        raise ValueError(f"{what}: targets must be a contiguous int32 tensor [{logits.shape[0]}]")
    if not 0 < scale < math.inf:
        raise ValueError(f"{what}: scale must be positive, not {scale}")


def _readable(logits: torch.Tensor):
    step, unit = logits.stride()
    rows, vocab = logits.shape
    if unit != 1 and vocab > 1:
        return K.contiguous(logits), vocab
    return logits, step if rows > 1 else vocab


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, scale: float = 1.0, ignore_index: int = -100) -> TokenLogProbs:
    """Of every row of scale * logits [rows, vocab] (row stride allowed; scale is 1 / temperature): the log-probability of its target, the entropy, and
    the `top` likeliest tokens (at most 32) with theirs; equal logits rank by index.  A target of ignore_index has log-probability 0, any other that is
    no token NaN.  Logits of -inf have probability 0; a row with NaN or +inf is NaN; one without anything above -inf has log-probabilities of
    -inf and entropy 0."""
    _check("token_logprobs", logits, targets, scale)
    rows, vocab = logits.shape
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"token_logprobs: 0 to {min(MAX_TOP, vocab)} alternatives, not {top}")
    _together("token_logprobs", logits, targets)
    if not logits.is_cuda:
        return _cpu(logits, targets, top, scale, ignore_index)
    f32 = dict(dtype=torch.float32, device=logits.device)
    out = TokenLogProbs(torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty((rows, 2), **f32), torch.empty((rows, top), **f32),
                        torch.empty((rows, top), dtype=torch.int32, device=logits.device))
    logits, step = _readable(logits)
    K._launch(N.require().oa_token_logprobs(K.dt(logits), logits.data_ptr(), step, targets.data_ptr(), *(t.data_ptr() for t in out), top, rows, vocab,
                                            float(scale), ignore_index, N.stream()), "oa_token_logprobs", outputs=(out.logprobs, out.entropy))
    return out


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
    _check("token_logprobs_backward", logits, targets, scale)
    rows, vocab = logits.shape
    for name, t, shape in (("dlogprobs", dlogprobs, (rows,)), ("dentropy", dentropy, (rows,)), ("result.entropy", result.entropy, (rows,)),
                           ("result.stats", result.stats, (rows, 2))):
        if t is not None and (t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous()):
            raise ValueError(f"token_logprobs_backward: {name} must be a contiguous float32 tensor {list(shape)}")
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype is not logits.dtype or (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
        raise ValueError(f"token_logprobs_backward: out must be {logits.dtype} {list(logits.shape)}, the elements of a row side by side, rows apart")
    _together("token_logprobs_backward", logits, targets, out, *(t for t in (dlogprobs, dentropy, result.entropy, result.stats) if t is not None))
    if not logits.is_cuda:
        return _backward_cpu(logits, targets, result, dlogprobs, dentropy, scale, ignore_index, out)
    logits, step = _readable(logits)
    K._launch(N.require().oa_token_logprobs_bwd(K.dt(logits), logits.data_ptr(), step, targets.data_ptr(), result.entropy.data_ptr(),
                                                result.stats.data_ptr(), N.ptr(dlogprobs), N.ptr(dentropy), out.data_ptr(),
                                                out.stride(0) if rows > 1 else vocab, rows, vocab, float(scale), ignore_index, N.stream()),
              "oa_token_logprobs_bwd", outputs=(out,))
    return out


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
