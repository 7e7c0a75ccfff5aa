"""Beam search's selection on both sides of its rules: how the bar is formed (up to 24 candidates, more; pieces
few and many for them) and how many pieces that reach it are read (4 n + 32) before the exact choice is
taken. Every choice has the definition's answer."""

import pytest
import torch

from tests.test_beam_gpu import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 23, 24, 25, 26, 63, 64])
@pytest.mark.parametrize("k,vocab", [(1, 2048 * 26), (2, 2048 * 14), (5, 2048 * 6 + 1), (3, 2048 * 100), (1, 2048 * 65 + 7), (8, 9000)])
def test_candidates_and_pieces(k, vocab, n):
    check(*inputs(2 * k, vocab, torch.float32, seed=n), k, n)


@pytest.mark.parametrize("n", [1, 2, 8, 24, 25, 64])
@pytest.mark.parametrize("more", [-1, 0, 1, 40])
def test_pieces_that_reach_the_bar(n, more):
    # Alike beams whose highest value stands in one token of as many pieces.
    k, pieces = 8, 60
    reach = 4 * n + 32 + more
    x, _ = inputs(1, 2048 * pieces, torch.float32, seed=n)
    x.clamp_(max=4.0)
    per = -(-reach // k)
    at = torch.arange(per, device="cuda") * 2048 + torch.randint(0, 2048, (per,), device="cuda", generator=torch.Generator("cuda").manual_seed(n))
    x = x.repeat(k, 1)
    for b in range(k):  # the first beams hold one more
        x[b, at[:reach // k + (b < reach % k)]] = 9.0
    # Beams of one number of such tokens tie; the others' totals lie apart.
    check(x, torch.full((k,), -12.0, device="cuda"), k, n)
    check(x.bfloat16(), torch.full((k,), -12.0, device="cuda"), k, n)
