"""Weight gradients over any number of rows: products whose operands both lie with the reduction down their rows, in bf16, against 64 bits."""
import pytest
import torch

from oa_b200 import _native as N
from oa_b200.ops import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(64, 104), (128, 128), (256, 256), (136, 1000), (1024, 512)])
@pytest.mark.parametrize("k", [1, 2, 7, 9, 63, 65, 127, 238, 1001, 4099])
def test_any_number_of_rows(m, n, k):
    """A sum of k products in 32 bits, each addition at most 2^-23 of the magnitudes so far (half of that rounded, all of it cut off), and the result's rounding.  The
    operands are the first rows of taller buffers whose other rows are NaN."""
    g = torch.Generator().manual_seed(m + n + k)
    tall = [torch.cat([torch.randn(k, c, generator=g), torch.full((70, c), float("nan"))]).bfloat16().cuda() for c in (m, n)]
    a, b = (t[:k] for t in tall)
    want = a.double().t() @ b.double()
    mag = a.double().abs().t() @ b.double().abs()
    sums = (k + 16) * 2.0 ** -23 * mag
    for out_dtype, u in ((torch.bfloat16, 2.0 ** -8), (torch.float32, 2.0 ** -24)):
        got = K.gemm(a, b, a_mn=True, b_mn=True, out_dtype=out_dtype)
        assert bool(((got.double() - want).abs() <= sums + u * (want.abs() + sums)).all())
        old = torch.randn(m, n, generator=g).to(out_dtype).cuda()
        got = K.gemm(a, b, a_mn=True, b_mn=True, out=old.clone(), accumulate=True)
        total = want + old.double()
        assert bool(((got.double() - total).abs() <= sums + 2.0 ** -23 * total.abs() + u * (total.abs() + sums)).all())
    K.check_status()


def test_rows_along_the_reduction_stay_whole():
    a, b = (torch.zeros(64, 16, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    with pytest.raises(N.OaKernelError):
        K.gemm(a[:, :9], b[:, :9])
