"""Reordering of beams whose pages are not in the pool: nothing is copied from them, as nothing is to them."""

import pytest
import torch

from babyvllm.kernels.beam import reorder_beams
from tests.test_beam_gpu import beams_case, check_reorder, reordered

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [-1, -(1 << 31), 1 << 29, None], ids=str)
@pytest.mark.parametrize("k", [2, 4, 8, 16, 32])
def test_a_parents_page_outside_the_pool_is_not_read(k, page):
    stack, tables, seq = beams_case(1, k, [20])
    page = stack.shape[2] if page is None else page  # the first behind the pool
    # The last beam's page is not there; the others take it, each other, or stay.
    parents = [k - 1] + [0 if b % 2 else b for b in range(1, k)]
    want, _ = reordered(stack, tables.clone(), seq, torch.tensor([[0] + parents[1:k - 1] + [k - 1]]))
    tables[k - 1, 1] = page
    before = tables.clone()
    parents[k - 1] = k - 1
    reorder_beams(list(stack.unbind(0)), tables, seq, torch.tensor([parents], device="cuda"))
    assert torch.equal(stack.cpu().view(torch.int16), want)
    assert torch.equal(tables[:, 1:], before[:, 1:]) and torch.equal(tables[0, :1], before[k - 1, :1])


@pytest.mark.parametrize("k", [3, 11, 32])
def test_pages_at_the_ends_of_the_pool(k):
    stack, tables, seq = beams_case(1, k, [23])
    tables[0, 1], tables[1, 1] = 0, stack.shape[2] - 1
    for b in range(2, k):
        tables[b, 1] = b
    check_reorder(stack, tables, seq, torch.tensor([[1, 0] + [b % 2 for b in range(2, k)]], device="cuda"))
