"""Commit, selection and reorder at the ends of what they take: caches past 2^31 elements and 2^32 bytes, calls on
another stream than the current one of their inputs' making, trees longer than the longest path."""

import random

import pytest
import torch

from babyvllm.kernels.beam import beam_select, reorder_beams
from babyvllm.kernels.tree_commit import commit_draft_tree
from tests import test_tree_commit_gpu as commit
from tests.test_beam_gpu import beams_case, inputs, reordered

pytestmark = pytest.mark.gpu
PAGES, HKV, D = 70000, 16, 128  # 4.6 GB a half


def behind(small):
    """A cache of PAGES pages whose last ones are those of `small` [2, n, 16, Hkv, D], and the first of them."""
    cache = torch.zeros(2, PAGES, *small.shape[2:], device="cuda", dtype=torch.bfloat16)
    first = PAGES - small.shape[1]
    assert first * small[0, 0].numel() > 1 << 31
    cache[:, first:] = small
    return cache, first


def test_commit_past_32_bits():
    rng = random.Random(4)
    specs = [commit.random_spec(rng, 20, 30, 1.0), commit.random_spec(rng, 7, 40, 0.9)]
    stack, md, draft, target, parents = commit.build(specs, layers=1, hkv=HKV, d=D)
    path, counts, answers, bits = commit.walk(specs, stack, md, 40)
    cache, first = behind(stack[0])
    md.block_tables = torch.where(md.block_tables >= 0, md.block_tables + first, -1).int()
    got = commit_draft_tree([cache], md, draft, target, parents)
    assert torch.equal(got[0].cpu(), path) and torch.equal(got[1].cpu(), counts)
    assert any(int(row[i]) > i for row, n in zip(path, counts) for i in range(int(n)))  # some rows move
    assert torch.equal(cache[:, first:].cpu().view(torch.int16), bits[0])
    assert not cache[:, :first].view(torch.int16).any()


def test_reorder_past_32_bits():
    stack, tables, seq = beams_case(2, 4, [37, 20], layers=1, hkv=HKV, d=D)
    beams = torch.tensor([[1, 2, 3, 0], [2, 2, 0, 0]], device="cuda")
    bits, _ = reordered(stack, tables, seq, beams)
    cache, first = behind(stack[0])
    reorder_beams([cache], tables + first, seq, beams)
    assert torch.equal(cache[:, first:].cpu().view(torch.int16), bits[0])
    assert not cache[:, :first].view(torch.int16).any()


def late(stream, tensors):
    """Zeros for now; the values come on `stream`, behind some milliseconds of other work."""
    values = [t.clone() for t in tensors]
    for t in tensors:
        t.zero_()
    torch.cuda.synchronize()
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(10):
            a = a @ a * 1e-4
        for t, v in zip(tensors, values):
            t.copy_(v)
    return values, a


def test_on_another_stream():
    side = torch.cuda.Stream()
    x, s = inputs(8, 32000)
    want = beam_select(x, s, 4, 8)
    kept = late(side, [x, s])
    with torch.cuda.stream(side):
        got = beam_select(x, s, 4, 8)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    rng = random.Random(6)
    specs = [commit.random_spec(rng, 20, 30, 1.0) for _ in range(4)]
    stack, md, draft, target, parents = commit.build(specs)
    path, counts, _, bits = commit.walk(specs, stack, md, md.max_query_len)
    kept = late(side, [stack, draft, target, parents])
    with torch.cuda.stream(side):
        got = commit_draft_tree(list(stack.unbind(0)), md, draft, target, parents)
    side.synchronize()
    assert torch.equal(got[0].cpu(), path) and torch.equal(got[1].cpu(), counts)
    assert torch.equal(stack.cpu().view(torch.int16), bits)

    stack, tables, seq = beams_case(2, 4, [37, 20])
    beams = torch.tensor([[1, 2, 3, 0], [2, 2, 0, 0]], device="cuda")
    bits, t = reordered(stack, tables, seq, beams)
    kept = late(side, [stack, tables, beams])
    with torch.cuda.stream(side):
        reorder_beams(list(stack.unbind(0)), tables, seq, beams)
    side.synchronize()
    assert torch.equal(tables.cpu(), t) and torch.equal(stack.cpu().view(torch.int16), bits)
    del kept


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
