"""Attention of drafted token trees on the GPU: against the formula in 64 bits, its masks and
refusals, its key ranges, graphs and streams.

Bounds. Weights w_j = p_j / sum p. The kernel rounds p_j to bf16 (off by at most 2^-8 of it)
before both products and sums the rounded values, so with d = 2^-8 + the scores' own error
(fp32 sums of D products and the exponent's rounding, under 2^-12 here) the output is off by at most
d / (1 - d) * sum_j w_j |v_j - o|, fp32 sums by n * 2^-24 * sum w|v|, the output's rounding by
2^-8 |o|. As a whole a row's errors of the weights are independent: their sum's norm is about
2^-8 / sqrt(3) * R, R^2 = sum_j w_j^2 |v_j - o|^2; 2 * 2^-8 * R + 2^-8 |o| is allowed, which a
missing or extra key of average weight exceeds below some 16,000 keys.
"""

import math
import random

import pytest
import torch

from babyvllm.kernels.tree_attn import ancestor_masks, paged_tree_attention
from babyvllm.worker.context import AttentionMetadata
from tests._cases import cdiv, python_path, scale_keys_by_position

pytestmark = pytest.mark.gpu
PAGE = 16


def random_tree(rng, n, branch=4):
    return [-1] + [rng.randrange(max(0, i - branch), i) for i in range(1, n)]


def build(specs, hkv, group, d, seed=0, words=None, fill=float("nan"), width_extra=0, q_view=False):
    """specs: (context, parents) per sequence; slots that hold no token are ``fill``."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads = hkv * group
    new = [len(p) for _, p in specs]
    ctx = [c for c, _ in specs]
    seq = [c + n for c, n in zip(ctx, new)]
    pages = [cdiv(n, PAGE) for n in seq]
    total, width = sum(pages) + 3, max(max(pages), 1) + width_extra
    cache = torch.full((2, total, PAGE, hkv, d), fill, device="cuda", dtype=torch.bfloat16)
    perm = torch.randperm(total, device="cuda", generator=g).tolist()
    tables, written = [], []
    for n, s in zip(pages, seq):
        t = [perm.pop() for _ in range(n)]
        written += [t[p // PAGE] * PAGE + p % PAGE for p in range(s)]
        tables.append(t + [-7 if i % 2 else 1 << 30 for i in range(width - n)])  # behind the row: never used
    if written:
        cache.view(2, -1, hkv, d)[:, torch.tensor(written, device="cuda")] = torch.randn(
            2, len(written), hkv, d, device="cuda", dtype=torch.bfloat16, generator=g)
    t = sum(new)
    if q_view:
        q = torch.randn(t, heads + 2 * hkv, d, device="cuda", dtype=torch.bfloat16, generator=g)[:, :heads]
    else:
        q = torch.randn(t, heads, d, device="cuda", dtype=torch.bfloat16, generator=g)
    qsl = [0]
    for n in new:
        qsl.append(qsl[-1] + n)
    mask, _ = ancestor_masks([p for _, p in specs], words)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    md = AttentionMetadata(torch.zeros(t, dtype=torch.int64, device="cuda"), i32(tables), i32(qsl), i32(seq), i32(ctx),
                           qsl, seq, ctx, max(new), max(seq), tree_mask=mask.cuda())
    return q, cache, md


def formula(q, cache, md, scale):
    """(outputs, elementwise bound, bound of a row's norm) in 64 bits on the CPU."""
    q64, mask = q.cpu().double(), md.tree_mask.cpu()
    c = cache.cpu().double()
    hkv, d = cache.shape[3], cache.shape[4]
    group = q.shape[1] // hkv
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape, 1e-30, dtype=torch.float64)
    row_tol = torch.full(q.shape[:2], 1e-30, dtype=torch.float64)
    qsl, tables = md.query_start_loc.tolist(), md.block_tables.tolist()
    for s, (ctx, n) in enumerate(zip(md.context_lens.tolist(), md.seq_lens.tolist())):
        a, b = qsl[s], qsl[s + 1]
        n = min(n, ctx + b - a, PAGE * len(tables[s]))
        pos = torch.arange(max(n, 0))
        page = torch.tensor(tables[s])[pos // PAGE]
        k, v = c[0][page, pos % PAGE], c[1][page, pos % PAGE]  # [n, Hkv, D]
        for r in range(a, b):
            sees = [p for p in range(n) if p < ctx or (int(mask[r, (p - ctx) // 64]) >> ((p - ctx) % 64)) & 1]
            if not sees:
                continue
            kk, vv = k[sees].repeat_interleave(group, 1), v[sees].repeat_interleave(group, 1)  # [m, H, D]
            score = (kk * q64[r]).sum(-1) * scale
            w = torch.softmax(score, 0)[..., None]
            o = (w * vv).sum(0)
            off = (vv - o).abs()
            bad = ~torch.isfinite(o)
            spread = (w * off).sum(0)
            reach = (w * vv.abs()).sum(0)
            dd = 2 ** -8 + 2 ** -12
            tol[r] += dd / (1 - dd) * spread + len(sees) * 2 ** -23 * reach + 2 ** -8 * o.abs()
            row_tol[r] += 2 * 2 ** -8 * (w * (vv - o)).norm(dim=-1).norm(dim=0) + 2 ** -8 * o.norm(dim=-1) \
                + len(sees) * 2 ** -23 * reach.norm(dim=-1)
            out[r] = o
            tol[r][bad] = math.inf
            row_tol[r][bad.any(-1)] = math.inf
    return out, tol, row_tol


def check(got, want):
    out, tol, row_tol = want
    got = got.cpu().double()
    fine = torch.isfinite(out)
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    assert torch.equal(got[~fine & ~torch.isnan(out)], out[~fine & ~torch.isnan(out)])
    diff = torch.where(fine, (got - out).abs(), torch.zeros_like(out))
    assert (diff <= tol).all(), f"off by up to {(diff / tol).max().item():.3g} times the bound"
    rows = diff.norm(dim=-1)
    assert (rows <= row_tol).all(), f"a row's norm is off by {(rows / row_tol).max().item():.3g} times the bound"


def run(q, cache, md, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    got = paged_tree_attention(q, cache, md, scale)
    check(got, formula(q, cache, md, scale))
    return got


_rng = random.Random(3)
SPECS = {
    "one_token": [(0, [-1])],
    "one_token_behind": [(1, [-1]), (15, [-1]), (16, [-1]), (31, [-1]), (32, [-1]), (33, [-1])],
    "steps": [(c, random_tree(_rng, n)) for c, n in ((0, 2), (1, 31), (15, 17), (16, 32), (17, 33), (31, 1), (32, 16), (63, 5))],
    "words": [(c, random_tree(_rng, n)) for c, n in ((40, 63), (7, 64), (0, 65), (100, 130), (33, 1))],
    "no_context": [(0, random_tree(_rng, n)) for n in (1, 7, 40, 100)],
    "ragged_and_empty": [(900, random_tree(_rng, 9)), (3, []), (0, random_tree(_rng, 20)), (0, []), (2100, [-1])],
    "forest": [(20, [-1, -1, 0, 1, -1, 4, 2]), (0, [-1, -1, -1])],
    "chains": [(c, list(range(-1, n - 1))) for c, n in ((500, 4), (64, 2), (127, 7), (0, 33))],
}
HEADS = [(4, 7, 128), (2, 7, 64), (1, 1, 128), (3, 2, 64), (1, 20, 64), (8, 4, 128)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("name", SPECS)
def test_against_the_formula(name, heads):
    run(*build(SPECS[name], *heads, seed=len(name)))


@pytest.mark.parametrize("ctx,n,heads", [(5000, 12, (2, 7, 64)), (3001, 70, (1, 7, 128)), (9000, 1, (1, 7, 128))])
def test_long_contexts(ctx, n, heads):
    run(*build([(ctx, random_tree(random.Random(ctx), n))], *heads, q_view=True, width_extra=5))


def test_many_sequences_of_mixed_lengths():
    rng = random.Random(9)
    run(*build([(rng.choice([0, 3, 50, 333, 1200]), random_tree(rng, rng.randint(1, 24))) for _ in range(70)], 2, 7, 64))


@pytest.mark.parametrize("heads", [(4, 7, 128), (2, 7, 64)], ids=str)
def test_python_path_gives_the_same_bits(monkeypatch, heads):
    q, cache, md = build(SPECS["ragged_and_empty"], *heads)
    got = run(q, cache, md)
    python_path(monkeypatch)
    assert torch.equal(paged_tree_attention(q, cache, md, q.shape[-1] ** -0.5), got)
    md.seq_lens_cpu = None  # no host lists: the table's width stands in
    check(paged_tree_attention(q, cache, md, q.shape[-1] ** -0.5), formula(q, cache, md, q.shape[-1] ** -0.5))


def raw_call(q, cache, md, scale, split, ranges):
    """The C entry with a choice of the context's ranges."""
    from babyvllm.kernels import _lib
    h = _lib.lib()
    t, heads, d = q.shape
    out = torch.full((t, heads, d), float("nan"), device="cuda", dtype=torch.bfloat16)
    ws = torch.full((max(4, h.bvllm_tree_workspace_bytes(t, heads, d, ranges) // 4),), float("nan"), device="cuda")
    bt, m, k = md.block_tables, md.tree_mask, cache[0]
    rc = h.bvllm_paged_tree_attention(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), cache[1].data_ptr(), *k.stride()[:3], cache.shape[1],
        bt.data_ptr(), bt.stride(0), bt.shape[1], md.query_start_loc.data_ptr(), md.seq_lens.data_ptr(),
        md.context_lens.data_ptr(), m.data_ptr(), m.stride(0), m.shape[1], scale, out.data_ptr(), out.stride(0),
        out.stride(1), md.seq_lens.shape[0], t, md.max_query_len, heads, cache.shape[3], d, 16, ws.data_ptr(), split,
        ranges, _lib.stream_handle(q.device))
    _lib.check(rc, "bvllm_paged_tree_attention")
    return out


@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64), (1, 3, 128), (1, 2, 64), (3, 2, 64), (12, 5, 128)], ids=str)
@pytest.mark.parametrize("split", [0, 1, 2, 3, 5, 12, 1000, -1, -2, -3, -5, -12, -1000])
def test_context_ranges_of_any_length(heads, split):
    # Contexts of no whole tile, of one, of several; blocks of 64 and of 128 columns.
    rng = random.Random(1)
    q, cache, md = build([(c, random_tree(rng, n)) for c, n in ((700, 9), (0, 3), (33, 40), (1500, 1), (64, 5), (127, 2))], *heads)
    want = formula(q, cache, md, 0.1)
    widest = max(1, cdiv(cdiv(md.block_tables.shape[1], 4), max(1, abs(split))))
    for ranges in sorted({1, 2, (widest + 1) // 2, widest} & set(range(1, widest + 1))):
        check(raw_call(q, cache, md, 0.1, split, ranges), want)


@pytest.mark.parametrize("heads", [(2, 7, 128), (4, 7, 64)], ids=str)
@pytest.mark.parametrize("seqs", [1, 3, 9, 20, 60, 64, 65, 140])
def test_every_number_of_waves_per_column(seqs, heads):
    rng = random.Random(seqs)
    specs = [(rng.choice([0, 5, 64, 100, 200]), random_tree(rng, rng.choice([1, 9, 30]))) for _ in range(seqs - 1)]
    q, cache, md = build(specs + [(130, random_tree(rng, 33))], *heads)
    want = formula(q, cache, md, 0.1)
    check(raw_call(q, cache, md, 0.1, 0, 0), want)
    check(raw_call(q, cache, md, 0.1, 1, 2), want)
    check(raw_call(q, cache, md, 0.1, -1, 2), want)


def test_masks_that_leave_rows_without_keys_or_without_themselves():
    q, cache, md = build([(0, [-1, 0, 0, 1]), (40, [-1, 0])], 2, 7, 64)
    md.tree_mask[1] = 0             # sees nothing
    md.tree_mask[2] = 1             # not itself
    md.tree_mask[3] = -1            # every drafted token, and bits of no token
    md.tree_mask[5] = 0             # the context alone
    got = run(q, cache, md)
    assert (got[1] == 0).all()


def test_seq_len_below_the_drafted_tokens_and_beyond_the_table():
    q, cache, md = build([(20, random_tree(random.Random(2), 30)), (100, [-1, 0]), (5, [-1])], 2, 7, 64)
    md.seq_lens[0] = 33             # tokens from 33 on are not in the cache
    md.seq_lens[1] = 60             # not even the whole context is
    md.seq_lens[2] = 0
    got = run(q, cache, md)
    assert (got[-1] == 0).all()
    # A row whose table is too short for it attends the keys that the table covers.
    q, cache, md = build([(100, [-1, 0, 0])], 2, 7, 64)
    md.block_tables = md.block_tables[:, :3].contiguous()
    run(q, cache, md)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64)], ids=str)
def test_what_a_row_does_not_see_does_not_reach_it(bad, heads):
    # Drafted tokens whose K and V are not finite spoil their own branch only.
    tree = [-1, 0, 0, 1, 2, 3, 4, 4, 6] + [0] * 30
    q, cache, md = build([(70, tree), (3, tree)], *heads)
    calls = (lambda: paged_tree_attention(q, cache, md, 0.1), lambda: raw_call(q, cache, md, 0.1, 1, 1))
    for s, ctx in enumerate((70, 3)):
        for node in (2, 6, 20):
            p = ctx + node
            page = int(md.block_tables[s, p // PAGE])
            cache[1, page, p % PAGE, :, node::3] = bad
            if node == 6:
                cache[0, page, p % PAGE, :, 0] = bad
    clean = cache.clone()
    clean[~torch.isfinite(clean)] = 0
    want = formula(q, clean, md, 0.1)
    mask = md.tree_mask.cpu()
    untouched = [r for r in range(q.shape[0]) if not any((int(mask[r, 0]) >> n) & 1 for n in (2, 6, 20))]
    assert len(untouched) > 60
    touched = [r for r in range(q.shape[0]) if (int(mask[r, 0]) >> 20) & 1]
    plain = torch.ones(heads[2], dtype=torch.bool)
    plain[20::3] = False  # the other dims of such a row are the formula's
    clean_v = cache.clone()
    clean_v[1][~torch.isfinite(clean_v[1])] = 0
    out, tol, _ = (w[touched] for w in formula(q, clean_v, md, 0.1))
    for call in calls:
        got = call().cpu()
        check(got[untouched], tuple(w[untouched] for w in want))
        assert len(touched) == 2 and not torch.isfinite(got[touched][..., 20::3]).any()
        assert ((got[touched].double() - out).abs()[..., plain] <= tol[..., plain]).all()


def test_scores_that_grow_and_scores_far_below_zero():
    q, cache, md = build([(900, [-1, 0, 0, 1]), (37, random_tree(random.Random(4), 50))], 2, 7, 64, fill=0.0)
    scale_keys_by_position(cache, md.block_tables, md.seq_lens, lambda p: 1 + p / 60)
    run(q, cache, md, 0.125)
    # A first visible key with a score of about -400: its weight is 1 all the same.
    q, cache, md = build([(0, [-1, -1, 1, 1] + [1] * 40)], 2, 7, 64, fill=0.0)
    q.copy_(torch.full_like(q, 4.0))
    cache[0].copy_(torch.full_like(cache[0], -12.0) + torch.randn_like(cache[0]) * 0.05)
    run(q, cache, md, 0.125)


def test_layouts_of_the_cache_and_of_q():
    q, cache, md = build(SPECS["ragged_and_empty"], 4, 7, 128)
    want = paged_tree_attention(q, cache, md, 0.09)
    head_major = cache.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)
    assert torch.equal(paged_tree_attention(q, head_major, md, 0.09), want)
    part = torch.cat([cache, cache.flip(0)], 1)[:, :cache.shape[1]]  # halves further apart
    assert torch.equal(paged_tree_attention(q, part, md, 0.09), want)
    wide = torch.zeros(q.shape[0], q.shape[1] + 3, 128, device="cuda", dtype=torch.bfloat16)
    wide[:, 2:2 + q.shape[1]] = q
    assert torch.equal(paged_tree_attention(wide[:, 2:2 + q.shape[1]], cache, md, 0.09), want)
    md.tree_mask = torch.cat([md.tree_mask, -torch.ones_like(md.tree_mask)], 1)  # words behind the tree
    assert torch.equal(paged_tree_attention(q, cache, md, 0.09), want)


def test_rows_behind_the_last_sequence_do_not_disturb():
    q, cache, md = build([(50, [-1, 0, 0]), (9, [-1])], 2, 7, 64)
    want = paged_tree_attention(q, cache, md, 0.125)
    more = torch.cat([q, torch.full_like(q, float("nan"))])
    md.tree_mask = torch.cat([md.tree_mask, -torch.ones_like(md.tree_mask)])
    assert torch.equal(paged_tree_attention(more, cache, md, 0.125)[:q.shape[0]], want)


def test_a_chain_is_a_prefill_and_one_token_a_decode():
    from babyvllm.kernels.paged_attn import paged_decode_attention
    from babyvllm.kernels.paged_prefill import paged_prefill_attention

    q, cache, md = build(SPECS["chains"], 4, 7, 128)
    want = formula(q, cache, md, 0.09)
    check(paged_tree_attention(q, cache, md, 0.09), want)
    check(paged_prefill_attention(q, cache, md, 0.09), want)
    q, cache, md = build([(c, [-1]) for c in (40, 0, 900, 16)], 4, 7, 128)
    want = formula(q, cache, md, 0.09)
    check(paged_tree_attention(q, cache, md, 0.09), want)
    check(paged_decode_attention(q, cache, md.block_tables, md.seq_lens, 0.09), want)


def test_in_a_graph_that_is_replayed_with_other_contents():
    rng = random.Random(5)
    specs = [[(c, random_tree(rng, n)) for c, n in ((cs, 7), (60, 20), (700, 3))] for cs in (1000, 5, 333)]
    sets = [build(s, 2, 7, 64, seed=i, fill=0.0) for i, s in enumerate(specs)]
    pool = max(c.shape[1] for _, c, _ in sets)
    width = max(md.block_tables.shape[1] for *_, md in sets)
    q = torch.zeros_like(sets[0][0])
    cache = torch.zeros(2, pool, *sets[0][1].shape[2:], device="cuda", dtype=torch.bfloat16)
    md = sets[0][2]
    md = AttentionMetadata(md.slot_mapping, torch.zeros(3, width, dtype=torch.int32, device="cuda"), md.query_start_loc,
                           md.seq_lens.clone(), md.context_lens.clone(), md.query_start_loc_cpu, [1024] * 3,
                           md.context_lens_cpu, md.max_query_len, 1024, tree_mask=md.tree_mask.clone())

    def load(i):
        sq, sc, sm = sets[i]
        q.copy_(sq)
        cache[:, :sc.shape[1]] = sc
        md.block_tables.zero_()
        md.block_tables[:, :sm.block_tables.shape[1]] = sm.block_tables
        for name in ("seq_lens", "context_lens", "tree_mask"):
            getattr(md, name).copy_(getattr(sm, name))

    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_tree_attention(q, cache, md, 0.125)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(paged_tree_attention(q, cache, md, 0.125))
        graphs.append(graph)
    for i in (0, 1, 2, 1, 0):
        load(i)
        eager = paged_tree_attention(q, cache, md, 0.125)
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
        check(eager, formula(q, cache, md, 0.125))


def test_on_another_stream():
    q, cache, md = build([(4000, random_tree(random.Random(6), 16))], 2, 7, 64)
    want = paged_tree_attention(q, cache, md, 0.125)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [paged_tree_attention(q, cache, md, 0.125) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_offsets_past_32_bits():
    # 40,000 pages of 64 KB a half: the last ones lie past 2^31 bytes and past 2^31 elements of the cache.
    hkv, d, pages = 16, 128, 40000
    cache = torch.zeros(2, pages, PAGE, hkv, d, device="cuda", dtype=torch.bfloat16)
    q, small, md = build([(50, [-1, 0, 0, 1])], hkv, 1, d, fill=0.0)
    want = paged_tree_attention(q, small, md, 0.09)
    n = small.shape[1]
    cache[:, pages - n:] = small
    md.block_tables = torch.where(md.block_tables < n, md.block_tables + (pages - n), 0).clamp(min=0).int()
    assert torch.equal(paged_tree_attention(q, cache, md, 0.09), want)


def test_no_memory_for_the_scratch_takes_the_whole_rows(monkeypatch):
    from babyvllm.kernels import _lib

    q, cache, md = build([(4000, random_tree(random.Random(6), 16))], 2, 7, 64)
    python_path(monkeypatch)
    assert _lib.lib().bvllm_tree_split_tiles(1, 16, 16, 14, 2, 64, md.block_tables.shape[1], 63, 63) != 0
    monkeypatch.setattr(_lib, "optional_scratch", lambda n, dev: None)
    run(q, cache, md)


def test_refusals():
    q, cache, md = build([(30, [-1, 0]), (4, [-1])], 2, 7, 64)
    from dataclasses import replace

    def refused(error, q=q, cache=cache, scale=0.1, **changes):
        with pytest.raises(error):
            paged_tree_attention(q, cache, replace(md, **changes), scale)

    refused(ValueError, tree_mask=None)
    refused(TypeError, q=q.float())
    refused(TypeError, cache=cache.half())
    refused(TypeError, tree_mask=md.tree_mask.int())
    refused(TypeError, seq_lens=md.seq_lens.long())
    refused(ValueError, tree_mask=md.tree_mask[:2])
    refused(ValueError, tree_mask=md.tree_mask[:, :0])
    refused(ValueError, max_query_len=65)
    refused(ValueError, block_tables=md.block_tables[:1])
    refused(ValueError, query_start_loc=md.query_start_loc[:2])
    refused(ValueError, context_lens=md.context_lens[:1])
    refused(ValueError, q=q.transpose(1, 2))
    refused(ValueError, cache=cache[0])
    refused(RuntimeError, tree_mask=md.tree_mask.cpu())
    refused(RuntimeError, q=q.cpu())
    for scale in (0.0, -0.1, float("nan"), float("inf")):
        refused(RuntimeError, scale=scale)
    refused(RuntimeError, q=torch.cat([q, q], 1)[:, :5])  # 5 query heads over 2
    refused(RuntimeError, cache=cache[:, :, :8].contiguous())  # pages of 8
    refused(ValueError, q=q[..., :32].contiguous())
    assert paged_tree_attention(q[:0], cache, md, 0.1).shape == (0, 14, 64)
