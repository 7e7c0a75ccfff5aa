"""Attention of drafted token trees on the GPU: values that are not finite in keys that every row sees, and
trees, contexts and numbers of ranges up to the largest.

The formula and its bounds are those of ``test_tree_attn_gpu``: an infinity or NaN in one dimension of a
visible key's V reaches that dimension of every row, and no other; in its K, the scores of its head.
"""

import random

import pytest
import torch

from babyvllm.kernels.tree_attn import paged_tree_attention
from tests.test_tree_attn_gpu import build, check, formula, random_tree, raw_call

pytestmark = pytest.mark.gpu
PAGE = 16
INF, NAN = float("inf"), float("nan")

# (context, position of the value): in whole steps of 32 keys, in the step that the context ends
# in, in its last key, in contexts of one and of whole steps.
PLACES = [(70, 3), (70, 40), (70, 63), (70, 64), (70, 66), (70, 69), (20, 0), (20, 19), (127, 95), (127, 96), (127, 126),
          (64, 63), (33, 32), (1, 0), (31, 30), (200, 191), (200, 192), (200, 199)]


def calls(q, cache, md):
    """The public call and every form of the C entry."""
    yield "public", paged_tree_attention(q, cache, md, 0.1)
    most = -(-md.block_tables.shape[1] // 4)
    for split, ranges in ((0, 0), (1, 1), (1, most), (-1, 1), (-1, most)):
        yield f"split {split}, {ranges} ranges", raw_call(q, cache, md, 0.1, split, ranges)


def spoil(cache, md, seq, pos, half, dim, value):
    """The value in one dimension of the key at `pos` of a sequence, every KV head."""
    page = int(md.block_tables[seq, pos // PAGE])
    cache[half, page, pos % PAGE, :, dim] = value


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64)], ids=str)
def test_context_values_that_are_not_finite_reach_their_dimension_of_every_row(heads, value):
    rng = random.Random(7)
    q, cache, md = build([(c, random_tree(rng, rng.choice([1, 3, 17, 40]))) for c, _ in PLACES], *heads)
    for s, (_, pos) in enumerate(PLACES):
        spoil(cache, md, s, pos, 1, (5 * s + pos) % heads[2], value)
    want = formula(q, cache, md, 0.1)
    rows, dims = (~torch.isfinite(want[0])).any(1).nonzero(as_tuple=True)
    assert len(rows) == q.shape[0] and len(set(dims.tolist())) > 10  # one dimension of each row
    for name, got in calls(q, cache, md):
        print(name, flush=True)
        check(got, want)


@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64)], ids=str)
def test_context_and_drafted_values_that_are_not_finite_in_one_step(heads):
    # Key 66 is seen by all; of the drafted ones some rows see the spoilt ones, others do not.
    tree = [-1, 0, 0, 1, 2, 3, 4, 4, 6] + [0] * 30
    q, cache, md = build([(70, tree), (20, tree), (96, tree)], *heads)
    for s, (ctx, pos) in enumerate(((70, 66), (20, 17), (96, 95))):
        spoil(cache, md, s, pos, 1, 9, INF)
        spoil(cache, md, s, ctx + 2, 1, 30, NAN)
        spoil(cache, md, s, ctx + 6, 1, 31, -INF)
        spoil(cache, md, s, ctx + 6, 1, 9, INF)
    want = formula(q, cache, md, 0.1)
    assert torch.isinf(want[0][..., 9]).all() and torch.isnan(want[0][..., 30]).any()
    for name, got in calls(q, cache, md):
        print(name, flush=True)
        check(got, want)


@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64)], ids=str)
def test_seq_len_below_the_context_with_values_that_are_not_finite(heads):
    # Only the first seq_len keys count: the spoilt one behind them does not.
    q, cache, md = build([(70, [-1, 0, 1]), (70, [-1, 0]), (90, [-1])], *heads)
    for s, (n, inside, behind) in enumerate(((68, 66, 69), (50, 49, 60), (64, 63, 64))):
        md.seq_lens[s] = n
        spoil(cache, md, s, inside, 1, 11, INF)
        spoil(cache, md, s, behind, 1, 12, NAN)
    want = formula(q, cache, md, 0.1)
    assert torch.isinf(want[0][..., 11]).all() and torch.isfinite(want[0][..., 12]).all()
    for name, got in calls(q, cache, md):
        print(name, flush=True)
        check(got, want)


@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64)], ids=str)
def test_context_keys_that_are_not_finite(heads):
    # A score of +inf or NaN leaves nothing but NaN of its row and head, one of -inf no weight of its key.
    rng = random.Random(8)
    for value in (INF, NAN):
        q, cache, md = build([(c, random_tree(rng, 9)) for c, _ in PLACES], *heads)
        for s, (c, pos) in enumerate(PLACES):
            if c > 1:
                spoil(cache, md, s, pos, 0, s % heads[2], value)
        want = formula(q, cache, md, 0.1)
        bad = torch.isnan(want[0])
        assert torch.equal(bad.any(-1), bad.all(-1)) and bad.any() and (value != value or not bad.all())
        for name, got in calls(q, cache, md):
            print(value, name, flush=True)
            check(got, want)


@pytest.mark.parametrize("heads", [(1, 2, 64), (1, 2, 128)], ids=str)
def test_trees_of_160_nodes(heads):
    rng = random.Random(160)
    q, cache, md = build([(c, random_tree(rng, n, b)) for c, n, b in ((0, 160, 4), (333, 160, 16), (90, 131, 1))], *heads)
    want = formula(q, cache, md, 0.1)
    for name, got in calls(q, cache, md):
        print(name, flush=True)
        check(got, want)


@pytest.mark.parametrize("heads", [(1, 3, 64), (1, 7, 128)], ids=str)
def test_a_context_of_32_thousand(heads):
    q, cache, md = build([(32011, random_tree(random.Random(32), 6))], *heads)
    check(paged_tree_attention(q, cache, md, 0.1), formula(q, cache, md, 0.1))


@pytest.mark.parametrize("split", [1, -1])
def test_every_number_of_ranges(split):
    q, cache, md = build([(1400, random_tree(random.Random(2), 12)), (640, [-1, 0])], 1, 7, 64)
    want = formula(q, cache, md, 0.1)
    for ranges in range(1, -(-md.block_tables.shape[1] // 4) + 1):
        check(raw_call(q, cache, md, 0.1, split, ranges), want)
