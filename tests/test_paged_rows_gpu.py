"""Paged attention around the limits of its kernels: rows of an item (8, 16 and more), keys that eight warps share, batches beyond 1024."""
import pytest
import torch

from oa_b200.ops import kernels as K

from test_paged import _check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,qh,kvh", [((1, 1, 1), 7, 1), ((1, 1, 1), 8, 1), ((1, 1, 1), 9, 1), ((2, 1, 2), 16, 2), ((1, 2, 1), 34, 4), ((3, 5, 4), 9, 3),
                                         ((1, 0, 1), 128, 1), ((4, 1, 0, 3), 4, 4)])
@pytest.mark.parametrize("prefix", [0, 15, 777])
def test_rows_around_the_limits(hd, rows, qh, kvh, prefix):
    if qh % kvh:
        qh -= qh % kvh
    _check_attention("cuda", torch.bfloat16, [max(600 * b + 13, f) for b, f in enumerate(rows)], list(rows), qh, kvh, hd, 16, prefix)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [16], [17], [33], [4097], [20011, 1, 3], [5, 9000, 0, 2, 130], [64] * 40, [1 + 37 * i % 500 for i in range(150)]])
def test_single_tokens_at_all_lengths(hd, ps, lens):
    _check_attention("cuda", torch.bfloat16, [max(n, 1) for n in lens], [1 if n else 0 for n in lens], 4, 2, hd, ps, 50 if len(lens) > 3 else 0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,prefix", [(2, 16389), (16, 4000), (17, 4000), (130, 2049)])
def test_a_long_prompt_for_few_and_many(hd, batch, prefix):
    _check_attention("cuda", torch.bfloat16, [1 + 29 * i % 90 for i in range(batch)], [1] * batch, 4, 4, hd, 64, prefix)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 32)])
def test_more_requests_than_the_sums_hold(dtype, hd):
    _check_attention("cuda", dtype, [1 + 7 * i % 40 for i in range(1100)], [1] * 1100, 2, 1, hd, 16, 33)


@pytest.mark.parametrize("hd", [64, 128])
def test_pieces_of_unequal_length_in_both_forms(hd):
    fresh = [40, 1, 0, 129, 7]
    lens = [f + 300 * (i % 3) for i, f in enumerate(fresh)]
    for prefix in (0, 130, 1000):                                 # five requests: each with the prompt's keys in its own items; twenty: the prompt once for all
        _check_attention("cuda", torch.bfloat16, lens, fresh, 8, 2, hd, 32, prefix)
        _check_attention("cuda", torch.bfloat16, [n % 200 + 24 for n in lens * 4], [f % 24 for f in fresh * 4], 8, 2, hd, 32, prefix)
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fresh,lens,prefix", [([700], [700], 0), ([300, 150], [300, 500], 200), ([513], [900], 129), ([260, 0], [260, 0], 1), ([1, 640], [1, 640], 77)])
def test_long_pieces_of_few_requests(hd, fresh, lens, prefix):
    _check_attention("cuda", torch.bfloat16, lens, fresh, 8, 2, hd, 16, prefix, room=5)
    _check_attention("cuda", torch.bfloat16, lens, fresh, 3, 3, hd, 128, prefix)
    K.check_status()


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("batch", [2048, 2049])
def test_the_most_requests_that_the_sums_hold_and_one_more(dtype, hd, batch):
    _check_attention("cuda", dtype, [1 + 5 * i % 23 for i in range(batch)], [1] * batch, 2, 1, hd, 16, 17)
