"""Sampling settings that are NaN: each keeps what its strictest number would, on both paths alike."""
import math

import pytest
import torch

from oa_b200.ops import sampling as S

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [40, 3000, 70000])
def test_settings_that_are_nan(device, vocab):
    x = torch.randn(4, vocab, generator=torch.Generator().manual_seed(vocab))
    x[:, 7] = x[:, 3] = 6.0                                       # two likeliest ones: the strictest min_p keeps both
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=device)  # noqa: E731
    nan = math.nan
    tokens, logprobs = S.sample(x.to(device), f([0.4, 0.6, 0.9, 0.9]), f([1.0, 1.0, 1.0, nan]), None, f([1.0, 1.0, nan, 1.0]), f([nan, nan, 0.0, 0.0]))
    assert tokens.tolist() == [3, 7, 3, 3]
    assert torch.allclose(logprobs.cpu(), torch.tensor([-math.log(2.0), -math.log(2.0), 0.0, 0.0]), rtol=2 ** -22, atol=0)
    tokens, _ = S.sample(x[:1].to(device), f([nan]), None, None, None, f([nan]))
    assert tokens.tolist() == [3]
