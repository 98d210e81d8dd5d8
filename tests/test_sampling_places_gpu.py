"""Sampling of rows that end inside a block's shared memory: places without a token hold nothing, whatever lay there before."""
import pytest
import torch

from oa_b200.ops import kernels as K
from oa_b200.ops import sampling as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 33, 255, 260, 500])
def test_short_rows_behind_long_ones_of_larger_logits(dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = 592
    x = torch.randn(rows, vocab, generator=g, device="cuda").to(dtype)
    large = torch.full((rows, 4000), 1e30, device="cuda", dtype=dtype)
    u, greedy = torch.rand(rows, generator=g, device="cuda"), torch.zeros(rows, device="cuda")
    want = torch.stack([(r == r.max()).nonzero()[0, 0] for r in x.float()])
    for _ in range(30):
        S.sample(large, u, greedy)
        tokens, logprobs = S.sample(x, u, greedy)
        assert torch.equal(tokens.long(), want) and bool((logprobs == 0).all())
    K.check_status()
