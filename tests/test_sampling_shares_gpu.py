"""Sampling at vocabularies around those at which a row goes to twice as many thread blocks."""
import pytest
import torch

from oa_b200.ops import kernels as K

from test_sampling import RULES, _check_on_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, v) for v in (25200, 25201, 25211, 26600, 50407, 100817, 201604, 201700)]
                         + [(torch.bfloat16, v) for v in (50400, 50405, 50421, 53100, 100825, 403250)])
def test_shares_about_half_of_a_multiprocessors_memory(dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rules = RULES * 11                                            # more rows than there are multiprocessors
    x = (torch.randn(len(rules), vocab, generator=g, device="cuda") * 2.5).to(dtype)
    _check_on_device(x, torch.rand(len(rules), generator=g, device="cuda"), rules)
    K.check_status()
