"""How many bits the softmax weights keep in the walk with masks of the draft tree attention.

Bound. A weight P enters the second product as two bf16 halves: the first is off by at most
2^-8 of P, the second by at most 2^-8 of that, so d = 2^-16 + the scores' own error (fp32 sums of
D <= 128 products of q and k, D * 2^-24 of their magnitudes, times the scale: under 2^-13 here, and the
exponent's roundings, under 2^-20 at these sizes). The output is off by at most d / (1 - d) *
sum_j w_j |v_j - o|, by fp32 sums, n * 2^-23 * sum_j w_j |v_j|, and by its own rounding, 2^-8 |o|.
With weights of one half (d = 2^-8) outputs near zero leave this bound, those of a few keys most often.
"""

import random

import pytest
import torch

from babyvllm.kernels.tree_attn import paged_tree_attention
from tests.test_tree_attn_gpu import build, random_tree, raw_call

pytestmark = pytest.mark.gpu
PAGE = 16


def bounded(q, cache, md, scale):
    """(outputs, bound) in 64 bits on the CPU."""
    q64, c, mask = q.cpu().double(), cache.cpu().double(), md.tree_mask.cpu()
    group = q.shape[1] // cache.shape[3]
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    tables, qsl = md.block_tables.tolist(), md.query_start_loc.tolist()
    d = 2 ** -16 + 2 ** -13 + 2 ** -20
    for s, (ctx, n) in enumerate(zip(md.context_lens.tolist(), md.seq_lens.tolist())):
        pos = torch.arange(n)
        page = torch.tensor(tables[s])[pos // PAGE]
        k, v = (h[page, pos % PAGE].repeat_interleave(group, 1) for h in (c[0], c[1]))  # [n, H, D]
        for r in range(qsl[s], qsl[s + 1]):
            sees = [p for p in range(n) if p < ctx or (int(mask[r, (p - ctx) // 64]) >> ((p - ctx) % 64)) & 1]
            kk, vv = k[sees], v[sees]
            magnitude = (kk * q64[r]).abs().sum(-1).max().item() * scale
            assert q.shape[2] * 2 ** -24 * magnitude < 2 ** -13
            w = torch.softmax((kk * q64[r]).sum(-1) * scale, 0)[..., None]
            o = (w * vv).sum(0)
            out[r] = o
            tol[r] = d / (1 - d) * (w * (vv - o).abs()).sum(0) + len(sees) * 2 ** -23 * (w * vv.abs()).sum(0) + 2 ** -8 * o.abs()
    return out, tol


def check(got, want):
    out, tol = want
    diff = (got.cpu().double() - out).abs()
    assert (diff <= tol).all(), f"off by up to {(diff / tol).max().item():.3g} times the bound"


SPECS = [(0, 5), (3, 9), (20, 33), (31, 1), (64, 17), (130, 40), (250, 8)]


@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64), (1, 1, 128), (3, 2, 64)], ids=str)
def test_one_launch(heads):
    rng = random.Random(21)
    q, cache, md = build([(c, random_tree(rng, n)) for c, n in SPECS], *heads)
    want = bounded(q, cache, md, 0.1)
    check(raw_call(q, cache, md, 0.1, 0, 0), want)
    check(paged_tree_attention(q[:5], cache, *first_sequence(md), 0.1), tuple(x[:5] for x in want))


def first_sequence(md):
    """The step of the first sequence alone: one launch, spread over the card."""
    from dataclasses import replace
    return (replace(md, block_tables=md.block_tables[:1], query_start_loc=md.query_start_loc[:2], seq_lens=md.seq_lens[:1],
                    context_lens=md.context_lens[:1], seq_lens_cpu=md.seq_lens_cpu[:1], tree_mask=md.tree_mask[:5],
                    max_query_len=5),)


@pytest.mark.parametrize("seqs", [1, 12, 40, 90])
@pytest.mark.parametrize("heads", [(2, 7, 64), (2, 7, 128)], ids=str)
def test_every_number_of_waves(heads, seqs):
    rng = random.Random(seqs)
    q, cache, md = build([(rng.choice([5, 40]), random_tree(rng, rng.choice([2, 9]))) for _ in range(seqs)], *heads)
    check(raw_call(q, cache, md, 0.1, 0, 0), bounded(q, cache, md, 0.1))


@pytest.mark.parametrize("split", [1, -1])
@pytest.mark.parametrize("heads", [(2, 7, 64), (2, 7, 128)], ids=str)
def test_keys_behind_the_whole_tiles(heads, split):
    # Contexts of no whole tile: ranges have none, and the keys behind them are all there are.
    rng = random.Random(22)
    q, cache, md = build([(c, random_tree(rng, n)) for c, n in ((63, 9), (0, 20), (40, 40))], *heads)
    check(raw_call(q, cache, md, 0.1, split, 1), bounded(q, cache, md, 0.1))
