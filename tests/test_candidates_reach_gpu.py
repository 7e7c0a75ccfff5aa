"""Commit of draft trees longer than the longest path that a call accepts."""

import pytest
import torch

from babyvllm.kernels.tree_commit import commit_draft_tree
from tests import test_tree_commit_gpu as commit

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nodes", [4095, 4096, 4097, 4500])
def test_trees_longer_than_the_longest_path(nodes):
    # A chain that is right to its end: the path holds 4096 nodes at most, also by default.
    spec = (5, list(range(-1, nodes - 1)), list(range(nodes)), list(range(1, nodes + 1)))
    stack, md, draft, target, parents = commit.build([spec], layers=1, hkv=1)
    bound = min(nodes, 4096)
    path, counts, answers, bits = commit.walk([spec], stack, md, bound)
    got = commit_draft_tree(list(stack.unbind(0)), md, draft, target, parents)
    assert torch.equal(got[0].cpu(), path) and got[1].item() == bound and got[2].item() == answers.item() == bound
    assert torch.equal(stack.cpu().view(torch.int16), bits)
