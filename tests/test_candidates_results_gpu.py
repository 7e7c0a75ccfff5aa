"""Results of the commit and of the beam selection as ordinary tensors: saved, copied and written to
without one showing in another, whichever of the wrappers' two host sides made them."""

import copy
import io

import pytest
import torch

from babyvllm.kernels.beam import beam_select
from babyvllm.kernels.tree_commit import commit_draft_tree
from tests import test_tree_commit_gpu as commit
from tests.test_beam_gpu import inputs
from tests._cases import python_path

pytestmark = pytest.mark.gpu


def committed():
    stack, md, draft, target, parents = commit.build([(3, [-1, 0, 1], [1, 2, 3], [2, 3, 9]), (20, [-1, 0], [4, 5], [5, 6])])
    return commit_draft_tree(list(stack.unbind(0)), md, draft, target, parents)


def selected():
    return beam_select(*inputs(6, 4000), 3, 5)


@pytest.mark.parametrize("python", [False, True], ids=["native", "python"])
@pytest.mark.parametrize("call", [committed, selected])
def test_results_are_tensors_of_their_own(call, python, monkeypatch):
    if python:
        python_path(monkeypatch)
    results = call()
    assert all(t.is_contiguous() and t.data_ptr() % t.element_size() == 0 for t in results)
    kept = [t.cpu() for t in results]
    file = io.BytesIO()
    torch.save(results, file)
    file.seek(0)
    for again in (torch.load(file, weights_only=True), copy.deepcopy(results), call()):
        assert all(torch.equal(a.cpu(), b) and a.dtype == b.dtype for a, b in zip(again, kept))
    for i, t in enumerate(results):  # written one after the other, the last first
        results[-1 - i].fill_(77)
        for j, u in enumerate(results):
            assert (u == 77).all() if j >= len(results) - 1 - i else torch.equal(u.cpu(), kept[j])
