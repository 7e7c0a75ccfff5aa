"""Attention of a sliding window and first tokens on the GPU: against the formula in 64 bits, what it does not
see, its cuts over work-groups, graphs and streams.

Bounds. Weights w_j = p_j / sum p. The kernels round p_j to bf16 (off by at most 2^-8 of it) before the
second product, and sum the rounded values (prompts) or those before (single rows): with d = 2^-8 + the
scores' own error (fp32 sums of D products and the exponent's rounding, under 2^-12 here) the output is off by
at most d / (1 - d) times sum_j w_j |v_j - o| or sum_j w_j |v_j|, fp32 sums by n * 2^-23 * sum w|v|, the
output's rounding by 2^-8 |o|. As a whole a row's errors of the weights are independent: their sum's norm is
about 2^-8 / sqrt(3) * R, R^2 = sum_j w_j^2 |v_j - o|^2 or sum_j w_j^2 |v_j|^2; 2 * 2^-8 * R + 2^-8 |o| is
allowed, which a missing or extra key of average weight exceeds below some 16,000 keys.
"""

import math
import random

import pytest
import torch

from babyvllm.kernels.window_attn import paged_window_attention
from babyvllm.worker.context import AttentionMetadata
from tests._cases import cdiv, python_path

pytestmark = pytest.mark.gpu
PAGE = 16
NAN, INF = float("nan"), float("inf")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def build(specs, hkv, group, d, window, sinks, seed=0, width_extra=0, q_view=False, rows_behind=0):
    """specs: (context, new tokens) per sequence. Slots that hold no token, and those of pages that no row of the
    sequence sees, hold NaN; table entries of the latter name a page of NaN or none at all."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads = hkv * group
    ctx, new = [c for c, _ in specs], [n for _, n in specs]
    seq = [c + n for c, n in specs]
    pages = [cdiv(n, PAGE) for n in seq]
    total, width = sum(pages) + 3, max(max(pages), 1) + width_extra
    cache = torch.full((2, total, PAGE, hkv, d), NAN, device="cuda", dtype=torch.bfloat16)
    perm = torch.randperm(total, device="cuda", generator=g).tolist()
    spare = perm.pop()
    tables, written = [], []
    for c, n, s in zip(ctx, pages, seq):
        first = max(0, c - window + 1) // PAGE
        t = []
        for i in range(n):
            page = perm.pop()
            if i < cdiv(sinks, PAGE) or i >= first:
                t.append(page)
                written += [page * PAGE + p % PAGE for p in range(i * PAGE, min(s, (i + 1) * PAGE))]
            else:
                t.append([spare, -1, 1 << 30, -2**31][i % 4])
        tables.append(t + [-7 if i % 2 else 1 << 30 for i in range(width - n)])
    if written:
        cache.view(2, -1, hkv, d)[:, torch.tensor(written, device="cuda")] = torch.randn(
            2, len(written), hkv, d, device="cuda", dtype=torch.bfloat16, generator=g)
    t = sum(new) + rows_behind
    if q_view:
        q = torch.randn(t, heads + 2 * hkv, d, device="cuda", dtype=torch.bfloat16, generator=g)[:, :heads]
    else:
        q = torch.randn(t, heads, d, device="cuda", dtype=torch.bfloat16, generator=g)
    qsl = [0]
    for n in new:
        qsl.append(qsl[-1] + n)
    md = AttentionMetadata(torch.zeros(t, dtype=torch.int64, device="cuda"), i32(tables), i32(qsl), i32(seq), i32(ctx),
                           qsl, seq, ctx, max(new), max(seq))
    return q, cache, md


def formula(q, cache, md, scale, window, sinks):
    """(outputs, elementwise bound, bound of a row's norm) in 64 bits. Rows behind the last sequence: not compared."""
    hkv, d = cache.shape[3], cache.shape[4]
    group, dev = q.shape[1] // hkv, q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    tol = torch.full(q.shape, 1e-30, dtype=torch.float64, device=dev)
    row_tol = torch.full(q.shape[:2], 1e-30, dtype=torch.float64, device=dev)
    qsl, tables = md.query_start_loc.tolist(), md.block_tables.tolist()
    num_pages = cache.shape[1]
    for s, (ctx, n) in enumerate(zip(md.context_lens.tolist(), md.seq_lens.tolist())):
        a, b = qsl[s], qsl[s + 1]
        n = min(n, ctx + b - a, PAGE * len(tables[s]))
        low = max(0, ctx - window + 1)
        pos = torch.tensor([p for p in range(max(n, 0)) if p < sinks or p >= low], dtype=torch.long, device=dev)
        if b == a or not len(pos):
            continue
        page = torch.tensor(tables[s], device=dev).long()[pos // PAGE].clamp(0, num_pages - 1)
        k, v = cache[0][page, pos % PAGE].double(), cache[1][page, pos % PAGE].double()  # [m, Hkv, D]
        for r in range(a, b, 8):
            at = ctx + torch.arange(r - a, min(b, r + 8) - a, device=dev)[:, None]
            sees = (pos <= at) & ((pos > at - window) | (pos < sinks))  # [rows, m]
            rows = slice(r, r + at.shape[0])
            for h in range(q.shape[1]):
                vv = v[:, h // group]
                score = (q[rows, h].double() @ k[:, h // group].T.contiguous()) * scale
                w = torch.nan_to_num(torch.softmax(score.masked_fill(~sees, -math.inf), -1), nan=NAN, posinf=INF)
                w = torch.where(sees.any(-1, keepdim=True), w, 0.0)[..., None]
                # (What a row does not see is left out, not multiplied by 0.)
                part = torch.where(sees[..., None], w * vv, 0.0)
                o = part.sum(1)
                off = torch.where(sees[..., None], vv - o[:, None], 0.0)
                reach = part.abs().sum(1)
                dd = 2 ** -8 + 2 ** -12
                m = sees.sum(-1)[:, None]
                spread = torch.maximum((w * off.abs()).sum(1), reach)
                norm = torch.maximum((w * off).norm(dim=-1).norm(dim=-1), part.norm(dim=-1).norm(dim=-1))
                out[rows, h] = o
                tol[rows, h] += dd / (1 - dd) * spread + m * 2 ** -23 * reach + 2 ** -8 * o.abs()
                row_tol[rows, h] += 2 * 2 ** -8 * norm + 2 ** -8 * o.norm(dim=-1) + m[:, 0] * 2 ** -23 * reach.norm(dim=-1)
    bad = ~torch.isfinite(out)
    tol[bad] = math.inf
    row_tol[bad.any(-1)] = math.inf
    end = qsl[-1]
    return tuple(x[:end].cpu() for x in (out, tol, row_tol))


def check(got, want):
    out, tol, row_tol = want
    got = got.cpu().double()[:out.shape[0]]
    fine = torch.isfinite(out)
    assert torch.equal(torch.isnan(got), torch.isnan(out)), (torch.isnan(got) != torch.isnan(out)).nonzero()[:4].tolist()
    assert torch.equal(got[~fine & ~torch.isnan(out)], out[~fine & ~torch.isnan(out)])
    diff = torch.where(fine, (got - out).abs(), torch.zeros_like(out))
    assert (diff <= tol).all(), f"off by up to {(diff / tol).max().item():.3g} times the bound"
    rows = diff.norm(dim=-1)
    assert (rows <= row_tol).all(), f"a row's norm is off by {(rows / row_tol).max().item():.3g} times the bound"


def raw_call(q, cache, md, scale, window, sinks, columns=128, split=0, runs=1, single=-1):
    """The C entry with a choice of blocks, of the ranges of their walks and of the runs of single rows."""
    from babyvllm.kernels import _lib
    h = _lib.lib()
    t, heads, d = q.shape
    seqs, hkv, bt, k = md.seq_lens.shape[0], cache.shape[3], md.block_tables, cache[0]
    runs = min(runs, bt.shape[1])
    # Every range that the table's keys can make, and fewer, where the last one takes what is left.
    ranges = cdiv(cdiv(bt.shape[1], 4), split) if split else 0
    ranges = max(1, ranges * 2 // 3) if split % 2 else ranges
    out = torch.full((t, heads, d), NAN, device="cuda", dtype=torch.bfloat16)
    ws = torch.full((max(4, h.bvllm_window_workspace_bytes(seqs, t, heads, d, ranges, runs) // 4),), NAN, device="cuda")
    rc = h.bvllm_paged_window_attention(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), cache[1].data_ptr(), *k.stride()[:3], cache.shape[1],
        bt.data_ptr(), bt.stride(0), bt.shape[1], md.query_start_loc.data_ptr(), md.seq_lens.data_ptr(),
        md.context_lens.data_ptr(), min(window, 2**31 - 1), min(sinks, 2**31 - 1), scale, out.data_ptr(), out.stride(0),
        out.stride(1), seqs, t, md.max_query_len, single, heads, hkv, d, 16, ws.data_ptr(), columns, split, ranges, runs,
        _lib.stream_handle(q.device))
    _lib.check(rc, "bvllm_paged_window_attention")
    return out


# Blocks of every width, whole and in ranges of a tile, of two and of three, single rows whole and in runs of a page and more.
FORMS = [(128, 0, 1), (64, 0, 2), (32, 0, 3), (128, 1, 1), (64, 1, 5), (32, 1, 1000), (128, 2, 1), (64, 3, 2), (32, 2, 1)]


def run(q, cache, md, window, sinks, scale=None, forms=()):
    """The public call, and the C entry's forms: all against the formula."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want = formula(q, cache, md, scale, window, sinks)
    got = paged_window_attention(q, cache, md, scale, window, sinks)
    check(got, want)
    for form in forms:
        print(window, sinks, form, flush=True)
        check(raw_call(q, cache, md, scale, window, sinks, *form), want)
    return got


_rng = random.Random(3)
SPECS = {
    "one_token": [(0, 1)],
    "rows": [(c, 1) for c in (0, 1, 14, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 200, 333, 1000)],
    "prompts": [(0, n) for n in (1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129, 190)],
    "behind": [(c, n) for c, n in ((1, 31), (15, 17), (16, 32), (17, 33), (31, 2), (63, 5), (64, 64), (100, 77), (300, 20))],
    "mixed_and_empty": [(900, 9), (3, 0), (0, 20), (500, 1), (0, 0), (77, 1), (210, 130), (0, 1)],
}
HEADS = [(4, 7, 128), (2, 7, 64), (1, 1, 128), (3, 2, 64), (1, 20, 64), (8, 1, 128)]
VIEWS = [(1, 0), (1, 1), (5, 3), (16, 0), (17, 4), (33, 16), (64, 40), (100, 4), (128, 64), (257, 1), (10**6, 0), (2**40, 2**40)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("name", SPECS)
def test_against_the_formula(name, heads):
    for i, (window, sinks) in enumerate(VIEWS):
        print(window, sinks, flush=True)
        run(*build(SPECS[name], *heads, window, sinks, seed=len(name)), window, sinks,
            forms=FORMS if name in ("behind", "mixed_and_empty") else FORMS[i % 3::3])


@pytest.mark.parametrize("specs,heads,window,sinks", [
    ([(9000, 1)], (2, 7, 64), 4096, 4), ([(5000, 1), (70, 1)], (1, 7, 128), 3001, 100), ([(20000, 40)], (1, 7, 128), 2500, 16),
    ([(6000, 130)], (1, 7, 64), 5000, 0), ([(0, 1500)], (1, 7, 128), 300, 4), ([(2000, 700), (4000, 1), (0, 300)], (1, 7, 64), 512, 33),
    ([(0, 600)], (1, 32, 64), 1000, 0), ([(3000, 1)] * 3, (1, 40, 128), 1024, 4),
], ids=str)
def test_long_sequences(specs, heads, window, sinks):
    run(*build(specs, *heads, window, sinks, q_view=True, width_extra=5), window, sinks, forms=[(128, 7, 4), (64, 16, 9), (32, 0, 1)])


def test_many_sequences_of_mixed_lengths():
    rng = random.Random(9)
    specs = [(rng.choice([0, 3, 50, 333, 1200]), rng.choice([1, 1, rng.randint(1, 40)])) for _ in range(130)]
    q, cache, md = build(specs, 2, 7, 64, 100, 4)
    run(q, cache, md, 100, 4, forms=FORMS)
    singles = sum(n == 1 for _, n in specs)
    check(raw_call(q, cache, md, 0.125, 100, 4, 64, 0, 1, singles), formula(q, cache, md, 0.125, 100, 4))
    check(raw_call(q, cache, md, 0.125, 100, 4, 64, 0, 1, 0), formula(q, cache, md, 0.125, 100, 4))  # in blocks too
    run(*build([(c, 1) for c, _ in specs], 2, 7, 64, 100, 20), 100, 20, forms=FORMS)


def test_rows_behind_the_last_sequence_are_left_as_they_are():
    for specs in ([(40, 1), (100, 1)], [(40, 9), (100, 1)]):
        q, cache, md = build(specs, 2, 7, 64, 30, 2, rows_behind=70)
        for form in FORMS:
            got = raw_call(q, cache, md, 0.1, 30, 2, *form)
            check(got, formula(q, cache, md, 0.1, 30, 2))
            assert torch.isnan(got[md.query_start_loc_cpu[-1]:]).all()


def test_rows_without_a_visible_key_give_zeros():
    q, cache, md = build([(300, 1), (40, 20), (0, 1), (200, 30)], 2, 7, 64, 20, 0)
    # Of the first sequence, nothing of what its row's window reaches is there; of the others, not all.
    md.seq_lens = i32([100, 45, 0, 0])
    md.seq_lens_cpu = md.seq_lens.tolist()
    got = run(q, cache, md, 20, 0, forms=FORMS)
    assert not got[0].any() and not got[21:].any() and got[1:5].any()
    md.block_tables = md.block_tables[:, :3].contiguous()  # and tables that end before the window
    run(q, cache, md, 20, 0, forms=FORMS)


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64), (4, 1, 64)], ids=str)
def test_values_that_are_not_finite_reach_the_rows_that_see_them(heads, value):
    window, sinks = 40, 3
    specs = [(c, n) for c, n in ((300, 1), (0, 90), (33, 50), (100, 130), (64, 1), (500, 3))]
    for half in (0, 1):
        q, cache, md = build(specs, *heads, window, sinks)
        for s, (c, n) in enumerate(specs):
            # A first token, keys in the window of some rows only, and the last one.
            for j, p in enumerate({1, max(0, c - 39), c + n // 2, c + n - 1}):
                page = int(md.block_tables[s, p // PAGE])
                if half:
                    cache[1, page, p % PAGE, :, (7 * s + 13 * j) % heads[2]] = value
                elif math.isnan(value):
                    cache[0, page, p % PAGE, 0, (7 * s + 13 * j) % heads[2]] = value
        run(q, cache, md, window, sinks, forms=FORMS)


def test_large_scores_and_weights_that_vanish():
    # Keys of one direction: the first rows' scores are far above or below the later ones'.
    for sign in (1, -1):
        q, cache, md = build([(200, 1), (0, 150), (120, 60)], 2, 7, 64, 50, 2)
        ramp = torch.linspace(0, 30, PAGE, device="cuda").to(torch.bfloat16)[None, :, None]
        cache[0, ..., 0] = sign * (ramp + torch.arange(cache.shape[1], device="cuda").to(torch.bfloat16)[:, None, None] % 7 * 30)
        q[..., 0] = 3.0
        want = formula(q, cache, md, 0.125, 50, 2)
        for form in FORMS:
            got = raw_call(q, cache, md, 0.125, 50, 2, *form).cpu().double()
            # (Scores of some thousands have errors of their own: 64 products of up to 630, 2^-24 each, a unit of the
            # exponent's 2^-13: weights off by at most 2^-10.)
            tol = want[1] + 2 ** -9 * want[1] * 2 ** 8
            assert ((got - want[0]).abs() <= tol).all()


def test_pages_past_2_31_elements():
    hkv, d, window = 8, 128, 64
    pages = 2**31 // (PAGE * hkv * d) + 40
    cache = torch.zeros(2, pages, PAGE, hkv, d, device="cuda", dtype=torch.bfloat16)
    table = i32([[3, pages - 1, 5, pages - 2, pages - 3, 7]])
    for p in table[0].tolist():
        cache[:, p] = torch.randn(2, PAGE, hkv, d, device="cuda", dtype=torch.bfloat16)
    for ctx, new in ((80, 1), (50, 40)):
        q = torch.randn(new, hkv * 2, d, device="cuda", dtype=torch.bfloat16)
        md = AttentionMetadata(None, table, i32([0, new]), i32([ctx + new]), i32([ctx]), [0, new], [ctx + new], [ctx], new, ctx + new)
        run(q, cache, md, window, 1, forms=FORMS[::2])


@pytest.mark.parametrize("kind", ["decode", "mixed"])
def test_captured_steps_replay_with_other_lengths(kind):
    new = [1] * 6 if kind == "decode" else [1, 30, 1, 1, 64, 7]
    longest = [700, 900, 400, 300, 500, 640]
    window, sinks = 100, 4
    q, cache, md = build([(c, n) for c, n in zip(longest, new)], 2, 7, 64, 10**6, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_window_attention(q, cache, md, 0.1, window, sinks)
        again = paged_window_attention(q, cache, md, 0.1, 33, 0)
    rng = random.Random(0)
    for _ in range(4):
        ctx = [rng.randint(0, c) for c in longest]
        md.context_lens.copy_(i32(ctx))
        md.seq_lens.copy_(i32([c + n for c, n in zip(ctx, new)]))
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        check(got, formula(q, cache, md, 0.1, window, sinks))
        check(again, formula(q, cache, md, 0.1, 33, 0))
        assert torch.equal(paged_window_attention(q, cache, md, 0.1, window, sinks), got)


def test_a_captured_step_takes_other_sequences():
    # One token of each but one sequence at first, prompts of all later: nothing of the captured step's host lists stays.
    q, cache, md = build([(300, 16)] * 6, 2, 7, 64, 10**6, 0)
    md.query_start_loc.copy_(i32([0, 1, 2, 3, 4, 20, 20]))
    md.query_start_loc_cpu, md.max_query_len = md.query_start_loc.tolist(), 96
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_window_attention(q, cache, md, 0.1, 100, 4)
    for new in ([16] * 6, [1] * 6, [91, 1, 1, 1, 1, 1], [0, 0, 96, 0, 0, 0], [1, 1, 1, 1, 16, 0]):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        md.query_start_loc.copy_(i32(starts))
        md.context_lens.copy_(i32([316 - n for n in new]))
        graph.replay()
        torch.cuda.synchronize()
        check(got, formula(q, cache, md, 0.1, 100, 4))


def test_on_two_streams_at_once():
    a = build([(3000, 1), (200, 1), (900, 1)], 2, 7, 64, 1000, 4)
    b = build([(100, 300), (2000, 1), (0, 64)], 2, 7, 64, 200, 4, seed=1)
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s, (case, out, (w, k)) in zip(streams, ((a, got[0], (1000, 4)), (b, got[1], (200, 4)))):
            with torch.cuda.stream(s):
                out.append(paged_window_attention(*case, 0.1, w, k))
    for s in streams:
        s.synchronize()
    for case, out, (w, k) in ((a, got[0], (1000, 4)), (b, got[1], (200, 4))):
        check(out[0], formula(*case, 0.1, w, k))
        assert all(torch.equal(o, out[0]) for o in out)


def test_the_python_path_and_absent_host_lists(monkeypatch):
    q, cache, md = build(SPECS["mixed_and_empty"], 2, 7, 64, 100, 4)
    got = run(q, cache, md, 100, 4)
    python_path(monkeypatch)
    assert torch.equal(paged_window_attention(q, cache, md, 0.125, 100, 4), got)
    md.query_start_loc_cpu = md.seq_lens_cpu = None
    check(paged_window_attention(q, cache, md, 0.125, 100, 4), formula(q, cache, md, 0.125, 100, 4))


def test_refusals():
    q, cache, md = build([(40, 1), (20, 9)], 2, 7, 64, 100, 4)
    call = lambda q=q, cache=cache, md=md, w=16, k=4: paged_window_attention(q, cache, md, 0.1, w, k)  # noqa: E731
    from dataclasses import replace
    with pytest.raises(TypeError):
        call(w=16.5)
    for w, k in ((0, 4), (-1, 4), (16, -1)):
        with pytest.raises(ValueError, match="window"):
            call(w=w, k=k)
    with pytest.raises(TypeError):
        call(q=q.float())
    with pytest.raises(TypeError):
        call(cache=cache.half())
    with pytest.raises(TypeError):
        call(md=replace(md, seq_lens=md.seq_lens.long()))
    with pytest.raises(ValueError):
        call(cache=cache[..., :32])
    with pytest.raises(ValueError):
        call(q=q.transpose(1, 2))
    with pytest.raises(ValueError):
        call(md=replace(md, block_tables=md.block_tables[:1]))
    with pytest.raises(ValueError):
        call(md=replace(md, query_start_loc=md.query_start_loc[:2]))
    with pytest.raises(RuntimeError, match="ROCm"):
        call(md=replace(md, context_lens=md.context_lens.cpu()))
