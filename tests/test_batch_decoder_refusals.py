"""OaBatchDecoder refuses what its operators do not take when it is made, not at its first step."""
import pytest
import torch

from oa_b200.core import fn_matrix as F
from oa_b200.models import OaGptConfig, OaGptModel
from oa_b200.serve import OaBatchDecoder


def _model(d_model, heads):
    return OaGptModel(OaGptConfig(64, d_model, 1, heads, 64, 96, "rms", "swiglu", 10000.0, False, 1e-5, 0.3))


def test_page_sizes():
    for size in (0, 8, 24, 256):
        with pytest.raises(ValueError, match="a page holds"):
            OaBatchDecoder(_model(32, 4), 2, 24, page_size=size)
    OaBatchDecoder(_model(32, 4), 2, 24, page_size=128)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_dims_of_the_kernels(dtype):
    prev = F.GetWeightDtype()
    F.SetWeightDtype(dtype)
    try:
        for d_model, heads in ((64, 4), (96, 1), (512, 2)):
            with pytest.raises(ValueError, match="heads of one of"):
                OaBatchDecoder(_model(d_model, heads), 2, 24, page_size=16)
        for d_model, heads in ((64, 2), (64, 1), (256, 2)):
            dec = OaBatchDecoder(_model(d_model, heads), 2, 24, page_size=16)
            assert len(dec.Generate([[1, 2], [3]], 3)[0]) == 3
    finally:
        F.SetWeightDtype(prev)
