"""A top-k whose cut lies further below the maximum than the bins of its first pass reach."""
import pytest
import torch

from oa_b200.ops import kernels as K

from test_sampling import _check, _check_on_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1.0, 10.0, 20.0, 100.0])
@pytest.mark.parametrize("near", [-31.96, -31.97, -31.98, -31.9845, -31.99, -32.0, -32.5])
def test_one_token_near_the_end_of_the_bins(temperature, near):
    """One maximum, one token about where the bins end, and all others beyond, more of them than a list holds."""
    x = torch.full((3, 20000), -33.0)
    x[:, 0] = 0.0
    x[0, 1] = near
    x[1, 1:700] = near
    x[2, 2:] -= torch.rand(19998, generator=torch.Generator().manual_seed(3))
    x[2, 1:9] = near
    _check("cuda", x, [0.5, 0.3, 0.8], [temperature] * 3, [1000] * 3, [1.0, 1.0, 0.9], [0.0] * 3)
    K.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,spread,part", [(32000, 2.5, 0.16), (50257, 10.0, 0.4), (201088, 10.0, 0.35), (201088, 8.0, 0.02)])
@pytest.mark.parametrize("peak", [0.0, 36.0])
def test_rows_that_spread_far(dtype, vocab, spread, part, peak):
    """The cut falls around 32 below the maximum, and the tokens there weigh something at the temperature."""
    g = torch.Generator(device="cuda").manual_seed(vocab + int(spread))
    rules = [(t, int(vocab * part) + i, p, 0.0) for i, (t, p) in enumerate([(5.0, 1.0), (10.0, 1.0), (30.0, 0.9), (100.0, 1.0), (1000.0, 0.99), (20.0, 0.5)] * 4)]
    x = torch.randn(len(rules), vocab, generator=g, device="cuda") * spread
    if peak:
        x[:, vocab // 3] = peak
    _check_on_device(x.to(dtype), torch.rand(len(rules), generator=g, device="cuda"), rules)
    K.check_status()


@pytest.mark.parametrize("k", [257, 400, 1000, 5000])
@pytest.mark.parametrize("masked", [-1e4, -40.0, -31.99])
def test_allowed_tokens_and_a_finite_mask(k, masked):
    """Tokens forbidden by a finite number: fewer and more of them allowed than top_k."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.full((6, 32000), masked, device="cuda")
    for r, n in enumerate((1, 100, k - 1, k, k + 1, 12000)):
        x[r, torch.randperm(32000, generator=g, device="cuda")[:n]] = torch.rand(n, generator=g, device="cuda") * 4
    _check_on_device(x, torch.rand(6, generator=g, device="cuda"), [(t, k, p, 0.0) for t, p in [(1.0, 1.0), (10.0, 0.9), (50.0, 1.0), (50.0, 0.99), (20.0, 1.0), (30.0, 0.7)]])
    K.check_status()
