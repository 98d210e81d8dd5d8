"""A step's `missing` is the number of its tokens without a slot, also for requests whose last page was not there when they came to it."""
import pytest
import torch

from oa_b200.ops import paged as P

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


@pytest.mark.parametrize("device", DEVICES)
def test_a_second_step_into_a_page_that_is_not_there(device):
    tables, free = torch.full((1, 4), -1, dtype=torch.int32, device=device), _i32([7], device)
    first = P.plan(_i32([0], device), _i32([20], device), tables, free, _i32([0], device), 16, 20)
    assert first.slots.tolist() == [112 + i for i in range(16)] + [-1] * 4 and first.missing.tolist() == [4]
    second = P.plan(first.lens, _i32([5], device), tables, free, first.taken, 16, 5)
    assert second.slots.tolist() == [-1] * 5 and second.missing.tolist() == [5] and second.taken.tolist() == [1]
    third = P.plan(second.lens, _i32([40], device), tables, _i32([7, 9, 3], device), second.taken, 16, 40)    # 7 to the end of the page, then two pages, one token over
    assert [s >= 0 for s in third.slots.tolist()] == [False] * 7 + [True] * 32 + [False] and third.missing.tolist() == [8]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batch,width,ps,pages,most", [(37, 5, 16, 90, 30), (300, 9, 16, 400, 12), (5, 3, 128, 6, 200), (64, 4, 32, 40, 1), (9, 2, 16, 0, 5)])
def test_missing_is_the_number_of_tokens_without_a_slot(device, batch, width, ps, pages, most):
    """Over many steps of a stack that runs out, with requests that end, some beyond their table's width, and rooms that are too small."""
    g = torch.Generator().manual_seed(batch)
    lens, tables = torch.zeros(batch, dtype=torch.int32, device=device), torch.full((batch, width), -1, dtype=torch.int32, device=device)
    free, taken = torch.randperm(pages, generator=g).to(torch.int32).to(device), _i32([0], device)
    ran_out = 0
    for i in range(14):
        fresh = torch.randint(0, most + 1, (batch,), generator=g).to(torch.int32)
        total = int(fresh.sum())
        step = P.plan(lens, fresh.to(device), tables, free, taken, ps, total)
        lost = int((step.slots < 0).sum())
        assert step.missing.tolist() == [lost]
        if total:                                                 # the same with less room for tokens: those beyond it are lost besides
            again = P.plan(lens, fresh.to(device), tables, free, taken, ps, total - 1)
            assert again.missing.tolist() == [lost + 1]
        ran_out += lost
        lens, taken = step.lens.clone(), step.taken
        if i % 3 == 2:
            taken = P.release((torch.rand(batch, generator=g) < 0.3).to(device), lens, tables, free, taken, ps)
    assert ran_out
