"""Sampling of rows that several thread blocks share: the ways on which top-p follows a top-k that ended without a list."""
import math

import pytest
import torch

from oa_b200.ops import kernels as K
from oa_b200.ops import sampling as S

from test_sampling import _check_on_device

pytestmark = pytest.mark.gpu


def _rows(seed, n, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, vocab, generator=g, device="cuda") * 2.5).to(dtype), torch.rand(n, generator=g, device="cuda")


def _check_again_and_again(x, u, rules, times=40):
    """The result is right, and the same while many rows are under way together."""
    _check_on_device(x, u, rules)
    f = lambda i, dtype=torch.float32: torch.tensor([r[i] for r in rules], dtype=dtype, device="cuda").repeat(8)  # noqa: E731
    wide, many = x.repeat(8, 1), u.repeat(8)
    args = (wide, many, f(0), f(1, torch.int32), f(2), f(3))
    first = S.sample(*args)
    for _ in range(times):
        for a, b in zip(S.sample(*args), first):
            assert torch.equal(a, b)
    K.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [9000, 50257, 201088])
def test_fewer_logits_than_top_k_and_then_top_p(dtype, vocab):
    """No more tokens than top_k are above -inf, so that nothing is cut before top-p."""
    x, u = _rows(vocab, 6, vocab, dtype)
    left = [1, 300, 301, 2000, 4000, 8191]
    for r, n in enumerate(left):
        x[r, torch.randperm(vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(r))[n:]] = -math.inf
    _check_again_and_again(x, u, [(1.0, max(n, 300), p, 0.0) for n, p in zip(left, [0.9, 0.5, 0.99, 0.8, 0.3, 0.95])])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [9000, 50257, 201088])
def test_a_top_k_among_equal_logits_and_then_top_p(dtype, vocab):
    """The cut of top-k falls among more equal logits than a list holds: masked by a finite number, or all alike."""
    x, u = _rows(vocab + 1, 5, vocab, dtype)
    x[0, 200:] = torch.finfo(dtype).min
    x[1] = 0.5
    x[2, 40:] = -1.0
    x[3] = (x[3] / 8).round() * 8
    x[4, vocab // 2:] = -30000.0
    _check_again_and_again(x, u, [(1.0, 1000, 0.9, 0.0), (0.8, 2000, 0.7, 0.0), (5.0, 3000, 0.9, 0.0), (20.0, 700, 0.6, 0.0), (3.0, vocab * 3 // 4, 0.95, 0.0)], 8)
