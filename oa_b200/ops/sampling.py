"""Sampling of next tokens from logits and given random numbers, on raw tensors.

CUDA tensors run csrc/kernels/sampling.cu, whose head states the rule in full; CPU tensors the plain statement of the same rule.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native as N
from . import kernels as K

MASS_BITS = 40      # a weight of 1 is this power of two: masses are whole numbers, so their sums do not depend on an order


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
           top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None):
    """One token for each row of logits [rows, vocab] (fp32 or bf16, row stride allowed) from u [rows] in [0, 1).

    Per row (tensors [rows], or None for off): logits over `temperature` (0 or less: the largest logit); of the `top_k` most likely
    tokens (0 or less: all) the fewest that together hold `top_p` of their probability (1 or more: all); of these the ones that have at
    least `min_p` of the likeliest one's probability.  The token is where u falls in what is kept, in the vocabulary's order.  Equal logits
    rank by index; the same inputs always give the same token.  Returns (tokens int32 [rows], log-probabilities fp32 [rows] among what
    was kept); (-1, -inf) for a row without a logit above -inf (NaN counts as -inf)."""
    if logits.dim() != 2 or u.dim() != 1 or u.numel() != logits.shape[0]:
        raise ValueError("sample: logits [rows, vocab] and one random number for each row")
    rows, vocab = logits.shape
    at = logits.get_device()
    for name, t, dtype in (("u", u, torch.float32), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is not None and (t.dtype is not dtype or t.numel() != rows or not t.is_contiguous() or t.get_device() != at):
            raise ValueError(f"sample: {name} must be a contiguous {dtype} tensor [{rows}] on {logits.device}")
    if not logits.is_cuda:
        return _sample_cpu(logits, u, temperature, top_k, top_p, min_p)
    step, unit = logits.stride()
    if vocab > 1 and unit != 1:
        logits, step = K.contiguous(logits), vocab
    tokens = torch.empty(rows, dtype=torch.int32, device=logits.device)
    logprobs = torch.empty_like(u)
    K._launch(N.require().oa_sample(K.dt(logits), logits.data_ptr(), step if rows > 1 else vocab, u.data_ptr(), N.ptr(temperature), N.ptr(top_k),
                                    N.ptr(top_p), N.ptr(min_p), tokens.data_ptr(), logprobs.data_ptr(), rows, vocab,
                                    K.status_word(logits.device).data_ptr(), N.stream()), "oa_sample")
    return tokens, logprobs


def _sample_cpu(logits, u, temperature, top_k, top_p, min_p):
    rows, vocab = logits.shape
    tokens = torch.full((rows,), -1, dtype=torch.int32)
    logprobs = torch.full((rows,), -float("inf"))
    for r in range(rows):
        x = logits[r].float()
        x = torch.where(x.isnan(), -float("inf"), x)
        if vocab == 0 or not bool((x > -float("inf")).any()):
            continue
        order = torch.sort(x, descending=True, stable=True).indices
        t = float(temperature[r]) if temperature is not None else 1.0
        if not t > 0:
            tokens[r], logprobs[r] = int(order[0]), 0.0
            continue
        top = x[order[0]]
        inv = 1.0 / temperature[r] if temperature is not None else torch.ones(())
        y = torch.where(x == top, 0.0, (x - top) * inv)
        w = torch.where(x == -float("inf"), 0.0, torch.exp(y))
        mass = (w * float(1 << MASS_BITS)).long()
        k = int(top_k[r]) if top_k is not None else 0
        order = order[:k] if k > 0 else order
        if top_p is not None and not float(top_p[r]) >= 1:
            m = mass[order]
            before = torch.cumsum(m, 0) - m
            n = int((before.double() < top_p[r].double() * m.sum().double()).sum())
            order = order[:max(n, 1)]
        keep = torch.zeros(vocab, dtype=torch.bool)
        keep[order] = True
        if min_p is not None:
            keep &= w >= torch.nan_to_num(min_p[r], nan=1.0).clamp(max=1.0)
        mass = torch.where(keep, mass, 0)
        total = int(mass.sum())
        at = float(u[r].double() * float(total))
        at = min(int(at), total - 1) if at > 0 else 0
        tokens[r] = int(torch.searchsorted(torch.cumsum(mass, 0), torch.tensor([at]), right=True))
        logprobs[r] = y[int(tokens[r])] - torch.log(torch.tensor(float(total), dtype=torch.float64) / float(1 << MASS_BITS)).float()
    return tokens, logprobs
