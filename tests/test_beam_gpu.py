"""Beam search's selection and the cache behind it on the GPU, against the definition in 64 bits.

Beams and tokens are equal to the definition's wherever its totals differ by more than the kernel's
can be off; inputs here are drawn so that no two totals at the border lie closer. A total is off by its
rounding to fp32 (2^-24 of it) and by the row's lse: fp32 terms (the exponent's argument and
result, 2^-23 each per unit of distance from the maximum, 16 at most where it weighs) and
fp32 sums of 32 and 64 terms: under 2^-18 of the sum, as absolute error of its logarithm."""

import random

import numpy as np
import pytest
import torch

from babyvllm.kernels.beam import beam_select, reorder_beams
from tests._cases import python_path

pytestmark = pytest.mark.gpu
PAGE = 16


def definition(logits, scores, k, n):
    x = logits.float().cpu().numpy().astype(np.float64)
    s = scores.cpu().numpy().astype(np.float64).reshape(-1)
    total = np.full(x.shape, -np.inf)
    for b, row in enumerate(x):
        if np.isfinite(s[b]) and not np.isnan(row).any() and np.isfinite(row.max()):
            top = row.max()
            total[b] = row + (s[b] - (top + np.log(np.exp(row - top).sum())))
    total = total.reshape(-1, k * x.shape[1])
    order = np.argsort(-total, axis=1, kind="stable")[:, :n]
    return np.take_along_axis(total, order, 1), order // x.shape[1], order % x.shape[1]


def check(logits, scores, k, n=None):
    n = min(2 * k, k * logits.shape[1]) if n is None else n
    got = beam_select(logits, scores, k, n)
    totals, beams, tokens = definition(logits, scores, k, n)
    assert np.array_equal(got[1].cpu().numpy(), beams) and np.array_equal(got[2].cpu().numpy(), tokens)
    s = got[0].cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isinf(s), np.isinf(totals))
    fin = np.isfinite(totals)
    assert (np.abs(s - totals)[fin] <= np.abs(totals[fin]) * 2 ** -24 + 2 ** -18).all()
    return got


def inputs(rows, vocab, dtype=torch.bfloat16, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * spread).to(dtype)
    return x, -torch.rand(rows, device="cuda", generator=g) * 4 - 10


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("groups,k,vocab", [(1, 1, 1), (1, 1, 5), (2, 3, 7), (3, 2, 64), (1, 32, 100), (2, 4, 2047), (2, 5, 2048),
                                            (1, 3, 2049), (4, 8, 4099), (1, 32, 50257), (2, 4, 151936), (3, 1, 20001)])
def test_against_the_definition(groups, k, vocab, dtype):
    check(*inputs(groups * k, vocab, dtype, seed=vocab), k)


@pytest.mark.parametrize("n", [1, 2, 7, 31, 64])
def test_numbers_of_candidates(n):
    check(*inputs(6, 9001, seed=n), 3, n)
    check(*inputs(2, 64, torch.float32, seed=n), 1, n)


def test_equal_logits_go_to_the_lowest_index():
    x, s = inputs(8, 6000)
    x.zero_()
    s.fill_(-3.0)
    got = check(x, s, 4, 16)
    assert (got[1] == 0).all() and torch.equal(got[2].cpu(), torch.arange(16).expand(2, 16))
    x[:, 5000:5100] = 1.0      # more equal ones than candidates, within one piece and beyond the first
    check(x, s, 4, 64)
    x[:, 1000:1003] = 1.0
    check(x, s, 4, 64)
    # Beams alike in all things: the first beam's tokens come first, whatever the row's alignment.
    y = torch.randn(1, 4097, device="cuda").bfloat16().expand(6, -1).contiguous()
    got = check(y, torch.full((6,), -1.5, device="cuda"), 3, 6)
    assert (got[1].cpu() == torch.tensor([0, 1, 2, 0, 1, 2])).all()


def test_few_values_among_many_tokens():
    x = torch.randint(-3, 4, (12, 30000), device="cuda").float()
    s = torch.arange(12, device="cuda").float() * -0.37
    check(x, s, 4, 64)
    check(x.bfloat16(), s, 6, 12)


def test_logits_in_order():
    # The best tokens all in one piece, more of them than candidates.
    x = torch.linspace(3, -3, 40000, device="cuda").expand(4, -1).contiguous()
    s = torch.tensor([-1.0, -2.5, -1.25, -9.0], device="cuda")
    check(x, s, 4, 64)
    check(x.flip(1).contiguous(), s, 2, 64)


def test_masked_vocabularies_and_beams_without_a_distribution():
    inf = float("inf")
    x, s = inputs(8, 9000, torch.float32)
    x[:, 100:] = -inf          # 100 allowed tokens
    x[:4, 5:] = -inf           # fewer than candidates
    check(x, s, 4, 64)
    s[1], s[2], s[5] = -inf, float("nan"), inf
    check(x, s, 4, 64)         # dead beams come last, with totals of -inf
    x[0, 17], x[3, 8999], x[4] = float("nan"), inf, -inf
    got = check(x, s, 4, 20)   # the first group has no live beam left: its first beam's first tokens
    assert (got[1][0] == 0).all() and (got[2][0] == torch.arange(20, device="cuda")).all()
    # A search's first step: one live beam.
    x, s = inputs(5, 3000, seed=4)
    s[1:] = -inf
    assert (check(x, s, 5, 10)[1] == 0).all()


@pytest.mark.parametrize("fill", [-float("inf"), torch.finfo(torch.bfloat16).min], ids=str)
@pytest.mark.parametrize("k,n,vocab,kept", [(4, 8, 151936, 20), (4, 8, 151936, 2), (4, 8, 151936, 1), (1, 64, 40000, 64),
                                            (1, 64, 40000, 63), (8, 9, 1000, 2), (3, 64, 70, 30)])
def test_masks_that_leave_more_or_fewer_tokens_than_candidates(k, n, vocab, kept, fill):
    x, s = inputs(2 * k, vocab, torch.float32, seed=kept)
    mask = torch.ones(2 * k, vocab, dtype=torch.bool, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for row in mask:
        row[torch.randperm(vocab, device="cuda", generator=g)[:kept]] = False
    x.masked_fill_(mask, fill)
    s[1::2] += 40.0  # other beams far ahead: their masked tokens' totals beat nothing
    check(x, s, k, n)
    check(x.bfloat16(), s, k, n)


def test_extreme_values():
    x, s = inputs(4, 5000, torch.float32, spread=1.0)
    x[0] *= 1e4
    x[1] *= 1e-6
    x[2, 77] = 3.0e38
    x[3, 1] = -3.4e38
    s.copy_(torch.tensor([-1e6, -8.0, -2.0, -7.5], device="cuda"))
    got = beam_select(x, s, 4, 8)
    totals, beams, tokens = definition(x, s, 4, 8)
    assert np.array_equal(got[1].cpu().numpy(), beams) and np.array_equal(got[2].cpu().numpy(), tokens)
    # Signed zeros are equal.
    z = torch.zeros(2, 300, device="cuda")
    z[:, ::2] = -0.0
    check(z, torch.tensor([-1.0, -1.0], device="cuda"), 2, 9)


@pytest.mark.parametrize("k,n,vocab", [(1, 2, 5000), (4, 8, 70000), (32, 64, 100), (32, 64, 4099), (32, 64, 50257), (2, 64, 30000)])
def test_scores_that_hide_logits(k, n, vocab):
    # At 1e20 a total's 64 bits step by 16384: all totals of equal scores are equal, and the
    # first tokens of the first beam lead.
    x, s = inputs(2 * k, vocab, seed=n)
    s.fill_(-1e20)
    scores, beams, tokens = beam_select(x, s, k, n)
    flat = torch.arange(n, device="cuda").expand(2, n)
    assert torch.equal(beams, flat // vocab) and torch.equal(tokens, flat % vocab)
    assert (scores == -1e20).all()
    # One beam far above the rest.
    s[k // 2] = 0.0
    s[k + k // 2] = 3e38
    check(x[:k].float(), s[:k], k, n)
    if vocab >= n:
        got = beam_select(x, s, k, n)
        assert (got[1] == k // 2).all() and (got[0][1] == 3e38).all()
        assert torch.equal(got[2][1], torch.arange(n, device="cuda"))


@pytest.mark.parametrize("groups,k,n,vocab,dtype", [(2, 32, 64, 100, torch.float32), (2, 32, 64, 4096, torch.bfloat16),
                                                    (1, 19, 38, 3000, torch.bfloat16), (2, 3, 64, 2500, torch.float32),
                                                    (2, 32, 64, 50257, torch.bfloat16), (3, 1, 64, 152064, torch.bfloat16)])
@pytest.mark.parametrize("kept", [None, 1, 40])
def test_many_candidates_among_equal_and_masked_ones(groups, k, n, vocab, dtype, kept):
    x, s = inputs(groups * k, vocab, torch.float32, seed=n + vocab)
    x = x.round().to(dtype)  # a few dozen distinct values
    if kept is not None:
        x[:, kept:] = -float("inf")
    s = s.round()
    scores, beams, tokens = beam_select(x, s, k, n)
    # Equal rows have equal bits; what is equal by the definition is equal here only within a beam:
    # the totals are the definition's, and no token is chosen twice or before an equal one.
    totals, _, _ = definition(x, s, k, n)
    got = scores.cpu().numpy().astype(np.float64)
    fin = np.isfinite(totals)
    assert np.array_equal(np.isinf(got), ~fin)
    assert (np.abs(got - totals)[fin] <= np.abs(totals[fin]) * 2 ** -24 + 2 ** -18).all()
    for g in range(groups):
        taken = list(zip(beams[g].tolist(), tokens[g].tolist()))
        assert len(set(taken)) == n
        for b in range(k):
            of_b = [t for beam, t in taken if beam == b]
            row = x[g * k + b].float()
            order = torch.argsort(-row.double(), stable=True)[:len(of_b)].tolist()
            assert of_b == order


def test_strided_rows_and_scores_of_any_shape():
    x, s = inputs(6, 4000, seed=8)
    want = check(x, s, 3, 6)
    for pad in (1, 8, 13):
        wide = torch.full((6, 4000 + pad), 9.0, device="cuda", dtype=torch.bfloat16)
        wide[:, pad:] = x
        got = beam_select(wide[:, pad:], s.view(2, 3), 3, 6)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    many = torch.stack([s, s + 1], 1)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x, many[:, 0], 3, 6), want))


@pytest.mark.parametrize("k,vocab,n", [(32, 524288, 64), (32, 524288, 9), (1, 3_000_001, 2), (1, 64, 64)])
def test_largest_and_smallest_sets_of_pieces(k, vocab, n):
    x, s = inputs(k, vocab, torch.float32 if vocab % 2 else torch.bfloat16, seed=n)
    x = x.float() + torch.rand_like(x, dtype=torch.float32) * 2 ** -9  # no ties
    totals = (s[:, None].double() + torch.log_softmax(x.double(), -1)).view(-1)
    want = totals.topk(n)
    got = beam_select(x, s, k, n)
    flat = got[1][0] * vocab + got[2][0]
    # (Equal fp32 logits are few among 16 million, but there: their order is by index.)
    assert torch.equal(totals[flat], want.values) and len(set(flat.tolist())) == n
    # Masked but for three tokens of every other beam: those, then the first masked ones.
    keep = torch.zeros_like(x, dtype=torch.bool)
    keep[::2, [3, vocab // 2, vocab - 1]] = True
    x[~keep] = -float("inf")
    x[1::2] = -float("inf")
    got = beam_select(x, s, k, n)
    flat = (got[1][0] * vocab + got[2][0]).tolist()
    live = min(n, 3 * ((k + 1) // 2))
    totals = torch.where(keep, s[:, None].double() + torch.log_softmax(x.double(), -1), -float("inf")).view(-1)
    order = totals.topk(live)
    assert torch.equal(totals[flat[:live]], order.values)
    rest = [i for i in range(min(n + 3, vocab)) if not keep.view(-1)[i]][:n - live]
    assert flat[live:] == rest and torch.isinf(got[0][0, live:]).all()


def test_one_row_for_all_beams(monkeypatch):
    # A search's first step: the prompt's logits for every beam, one of them live.
    x, s = inputs(4, 5000)
    s[1:] = -float("inf")
    want = check(x[:1].expand(4, -1), s, 4)
    for got in (beam_select(x[:1].repeat(4, 1), s, 4), beam_select(x[:1].expand(4, -1), s, 4, 8)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    python_path(monkeypatch)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x[:1].expand(4, -1), s, 4), want))


def test_defaults_the_python_path_and_no_rows(monkeypatch):
    x, s = inputs(6, 4000)
    want = beam_select(x, s, 3, 6)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x, s, 3), want))
    python_path(monkeypatch)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x, s, 3, 6), want))
    assert [t.shape for t in beam_select(x[:0], s[:0], 3)] == [(0, 6)] * 3
    assert beam_select(x[:2, :1], s[:2], 2)[0].shape == (1, 2)


def test_select_in_a_graph():
    x, s = inputs(8, 32000)
    beam_select(x, s, 4, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam_select(x, s, 4, 8)
    for seed in (1, 2, 3, 1):
        y, t = inputs(8, 32000, seed=seed)
        x.copy_(y), s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, beam_select(y, t, 4, 8)))


def test_select_refusals():
    x, s = inputs(6, 400)

    def refused(error, *args):
        with pytest.raises(error):
            beam_select(*args)

    refused(RuntimeError, x.cpu(), s.cpu(), 3)
    refused(RuntimeError, x, s.cpu(), 3)
    refused(TypeError, x.half(), s, 3)
    refused(TypeError, x, s.double(), 3)
    refused(ValueError, x.t(), s, 3)
    refused(ValueError, x[0], s, 3)
    refused(ValueError, x, s, 4)
    refused(ValueError, x, s, 0)
    refused(ValueError, x, s[:5], 3)
    refused(ValueError, x, s, 3, 0)
    refused(ValueError, x, s, 3, 65)
    refused(ValueError, x[:, :2], s, 3, 7)
    refused(ValueError, torch.cat([x] * 11), torch.cat([s] * 11), 33)
    wide = torch.zeros(32, 600_000, device="cuda", dtype=torch.bfloat16)
    refused(RuntimeError, wide, torch.zeros(32, device="cuda"), 32, 4)  # more pieces than a group may have


# ------------------------------------------------------------------ the cache


def beams_case(groups, k, lens, layers=3, hkv=2, d=64, seed=0, width_extra=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(lens) // PAGE + 1 + width_extra
    total = groups * k * width + 5
    tables = torch.randperm(total, device="cuda", generator=g)[:groups * k * width].view(groups * k, width).int()
    stack = torch.randint(-32768, 32768, (layers, 2, total, PAGE, hkv, d), device="cuda", dtype=torch.int16,
                          generator=g).view(torch.bfloat16)
    seq = torch.tensor([n for n in lens for _ in range(k)], dtype=torch.int32, device="cuda")
    return stack, tables, seq


def reordered(stack, tables, lens, beams):
    bits, t = stack.cpu().view(torch.int16).clone(), tables.cpu().clone()
    old, old_t = bits.clone(), t.clone()
    groups, k = beams.shape
    for g in range(groups):
        n = int(lens[g * k])
        for b in range(k):
            p = int(beams[g, b])
            if not 0 <= p < k:
                continue
            full = min(max(n, 0) // PAGE, t.shape[1])
            t[g * k + b, :full] = old_t[g * k + p, :full]
            if n > 0 and full < t.shape[1]:
                to, frm = int(old_t[g * k + b, full]), int(old_t[g * k + p, full])
                bits[:, :, to, :n % PAGE] = old[:, :, frm, :n % PAGE]
    return bits, t


def check_reorder(stack, tables, lens, beams):
    bits, t = reordered(stack, tables, lens, beams)
    assert reorder_beams(list(stack.unbind(0)), tables, lens, beams) is tables
    assert torch.equal(tables.cpu(), t)
    assert torch.equal(stack.cpu().view(torch.int16), bits)


@pytest.mark.parametrize("k", [1, 2, 4, 5, 8, 16, 17, 32])
def test_random_parents(k):
    rng = random.Random(k)
    lens = [0, 1, 15, 16, 17, 31, 200, 1003]
    case = beams_case(len(lens), k, lens, seed=k)
    beams = torch.tensor([[rng.randrange(k) for _ in range(k)] for _ in lens], device="cuda")
    check_reorder(*case, beams)


def test_swaps_cycles_and_one_parent_for_all():
    for beams in ([[1, 0, 3, 2]], [[1, 2, 3, 0]], [[2, 2, 2, 2]], [[0, 1, 2, 3]], [[-1, 0, 4, 1 << 40]]):
        check_reorder(*beams_case(1, 4, [77]), torch.tensor(beams, device="cuda"))


@pytest.mark.parametrize("hkv,d,layers", [(4, 128, 5), (1, 64, 70), (3, 128, 1)])
def test_shapes_of_the_cache(hkv, d, layers):
    beams = torch.tensor([[3, 0, 0, 2], [1, 1, 2, 0]], device="cuda")
    check_reorder(*beams_case(2, 4, [29, 45], layers=layers, hkv=hkv, d=d), beams)


def test_wide_tables_full_tables_and_views(monkeypatch):
    beams = torch.tensor([[1, 2, 0]], device="cuda")
    check_reorder(*beams_case(1, 3, [9000], layers=1, hkv=1), beams)           # more columns than a work-group
    stack, tables, seq = beams_case(1, 3, [64], width_extra=-1)                # every page full, none behind
    check_reorder(stack, tables, seq, beams)
    seq.fill_(200)                                                            # longer than the table
    check_reorder(stack, tables, seq, beams)
    stack, tables, seq = beams_case(2, 3, [50, 33])
    wide = torch.zeros(6, tables.shape[1] + 7, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + tables.shape[1]] = tables
    check_reorder(stack, wide[:, 3:3 + tables.shape[1]], seq, torch.cat([beams, beams]))
    assert (wide[:, :3] == 0).all() and (wide[:, -4:] == 0).all()
    python_path(monkeypatch)
    check_reorder(stack, tables.clone(), seq, torch.cat([beams, beams]))
    t = tables.clone()
    want = reordered(stack, t, seq, torch.cat([beams, beams]))[1]
    assert torch.equal(reorder_beams([], t, seq, torch.cat([beams, beams])).cpu(), want)  # the tables alone


def test_pages_outside_the_pool_are_not_written():
    stack, tables, seq = beams_case(1, 3, [20])
    tables[1, 1] = -3
    tables[2, 1] = 1 << 29
    before = stack.clone()
    reorder_beams(list(stack.unbind(0)), tables, seq, torch.tensor([[0, 0, 0]], device="cuda"))
    assert torch.equal(stack.view(torch.int16), before.view(torch.int16))


def test_reorder_in_a_graph():
    stack, tables, seq = beams_case(2, 4, [37, 120])
    first_stack, first_tables = stack.clone(), tables.clone()
    beams = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    caches = list(stack.unbind(0))
    reorder_beams(caches, tables, seq, beams)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_beams(caches, tables, seq, beams)
    stack.copy_(first_stack), tables.copy_(first_tables)
    for p in ([[1, 0, 3, 2], [0, 0, 1, 1]], [[3, 3, 3, 0], [2, 1, 0, 3]], [[0, 0, 0, 0], [1, 2, 3, 0]]):
        beams.copy_(torch.tensor(p))
        bits, t = reordered(stack, tables, seq, beams)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tables.cpu(), t) and torch.equal(stack.cpu().view(torch.int16), bits)


def test_reorder_refusals():
    stack, tables, seq = beams_case(2, 3, [20, 40])
    caches, beams = list(stack.unbind(0)), torch.zeros(2, 3, dtype=torch.int64, device="cuda")

    def refused(error, caches=caches, tables=tables, seq=seq, beams=beams):
        with pytest.raises(error):
            reorder_beams(caches, tables, seq, beams)

    refused(RuntimeError, tables=tables.cpu())
    refused(RuntimeError, beams=beams.cpu())
    refused(RuntimeError, caches=[caches[0].cpu()])
    refused(TypeError, tables=tables.long())
    refused(TypeError, beams=beams.int())
    refused(TypeError, caches=[caches[0].half()])
    refused(ValueError, beams=beams.view(-1))
    refused(ValueError, beams=torch.zeros(1, 33, dtype=torch.int64, device="cuda"))
    refused(ValueError, tables=tables[:5])
    refused(ValueError, tables=tables[:1].expand(6, -1))
    refused(ValueError, seq=seq[:5])
    refused(ValueError, caches=[caches[0], caches[1][:, :2]])
    refused(ValueError, caches=[caches[1], caches[0], caches[1]])
    refused(RuntimeError, caches=[c[:, :, :8].contiguous() for c in caches])
