"""The cache calls of draft trees and beams while other threads change the list of caches that they were
given: a call takes the caches that were in the list when it began."""

import threading

import pytest
import torch

from babyvllm.kernels.beam import reorder_beams
from babyvllm.kernels.tree_commit import commit_draft_tree
from tests import test_tree_commit_gpu as commit
from tests.test_beam_gpu import beams_case

pytestmark = pytest.mark.gpu


def changed_meanwhile(caches, call, calls=400):
    """`calls` calls on a list that another thread empties and fills again; the exceptions of both."""
    given, errors, done = list(caches), [], threading.Event()

    def change():
        try:
            while not done.is_set():
                given.clear()
                given.extend(caches)
                given[:] = caches[:1]
                given[:] = caches
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    other = threading.Thread(target=change)
    other.start()
    try:
        for _ in range(calls):
            call(given)
    finally:
        done.set()
        other.join()
    torch.cuda.synchronize()
    return errors


def test_commit():
    specs = [(3, [-1, 0, 1], [1, 2, 3], [2, 3, 9]), (20, [-1, 0, 0], [4, 6, 5], [5, 6, 7])]
    stack, md, draft, target, parents = commit.build(specs, layers=30)
    path, counts, answers, _ = commit.walk(specs, stack, md, 3)

    def call(caches):
        got = commit_draft_tree(caches, md, draft, target, parents)
        assert all(a.shape == b.shape for a, b in zip(got, (path, counts, answers)))
        results.append(got)

    results = []
    assert changed_meanwhile(list(stack.unbind(0)), call) == []
    for got in results:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, (path, counts, answers)))


def test_reorder():
    stack, tables, seq = beams_case(2, 4, [37, 20], layers=30)
    beams = torch.tensor([[0, 0, 2, 2], [1, 1, 3, 3]], device="cuda")  # the same again after the first
    first = reorder_beams(list(stack.unbind(0)), tables, seq, beams).clone()
    want = stack.clone()
    assert changed_meanwhile(list(stack.unbind(0)), lambda caches: reorder_beams(caches, tables, seq, beams)) == []
    assert torch.equal(tables, first) and torch.equal(stack.view(torch.int16), want.view(torch.int16))
