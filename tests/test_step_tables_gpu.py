"""Block tables and slot maps from request lengths on the GPU, against lists built one entry at a time.

All results are whole numbers: they have to be equal.
"""

import random

import pytest
import torch

from babyvllm.kernels.step_tables import StepTables, build_step_tables

pytestmark = pytest.mark.gpu
PAGE = 16


def held_entries(ctx, new, window, sinks):
    """Table entries that a request holds pages for."""
    pages = -(-(ctx + new) // PAGE)
    if window is None:
        return list(range(pages))
    first = max(0, ctx - window + 1) // PAGE
    return [i for i in range(pages) if i * PAGE < sinks or i >= first]


def formula(new, ctx, pages, rows, width, window=None, sinks=0, pad_page=0):
    new, ctx = [max(n, 0) for n in new], [max(c, 0) for c in ctx]
    tables, qsl, positions, slots, taken = [], [0], [], [], 0
    for n, c in zip(new, ctx):
        page_of = {}
        for i in held_entries(c, n, window, sinks):
            page_of[i] = pages[taken] if taken < len(pages) else None
            taken += 1
        tables.append([pad_page if page_of.get(i) is None else page_of[i] for i in range(width)])
        qsl.append(min(qsl[-1] + n, rows))
        for p in range(c, c + n)[:qsl[-1] - qsl[-2]]:
            page = page_of.get(p // PAGE) if p // PAGE < width else None
            positions.append(p)
            slots.append(-1 if page is None or page < 0 else page * PAGE + p % PAGE)
    pad = rows - len(positions)
    return StepTables(torch.tensor(tables, dtype=torch.int32).view(len(new), width),
                      torch.tensor(qsl, dtype=torch.int32),
                      torch.tensor([n + c for n, c in zip(new, ctx)], dtype=torch.int32),
                      torch.tensor(positions + [0] * pad, dtype=torch.int64),
                      torch.tensor(slots + [-1] * pad, dtype=torch.int64))


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(got, want):
    for name, g, w in zip(StepTables._fields, got, want):
        assert g.dtype == w.dtype and g.shape == w.shape, name
        assert torch.equal(g.cpu(), w), (name, (g.cpu() != w).nonzero()[:5].tolist())


def both(new, ctx, rows, width, **k):
    rng = random.Random(1)
    n = sum(len(held_entries(max(c, 0), max(x, 0), k.get("window"), k.get("sinks", 0))) for x, c in zip(new, ctx))
    pages = list(range(n))
    rng.shuffle(pages)
    check(build_step_tables(i32(new), i32(ctx), i32(pages), rows, width, **k), formula(new, ctx, pages, rows, width, **k))


@pytest.mark.parametrize("new,ctx,rows,width", [
    ([1], [0], 1, 1), ([1], [15], 1, 1), ([1], [16], 1, 2), ([17], [0], 17, 2), ([16], [16], 16, 2),
    ([0], [0], 0, 1), ([0], [33], 4, 5), ([0, 1, 0], [7, 31, 0], 3, 4), ([5, 1, 40], [0, 100, 3], 46, 7),
    ([5, 1, 40], [0, 100, 3], 64, 30), ([], [], 0, 3), ([], [], 5, 3),
], ids=str)
def test_small_steps(new, ctx, rows, width):
    both(new, ctx, rows, width)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (15, 0), (16, 4), (17, 16), (64, 17), (33, 1000), (2**31 - 1, 2**31 - 1),
                                          (2**40, 2**40), (100, 0)])
def test_windowed_requests_hold_what_their_rows_see(window, sinks):
    ctx = [0, 1, 14, 15, 16, 17, 31, 32, 33, 63, 64, 65, 79, 80, 81, 200, 1000, 1001]
    new = [1, 0, 2, 1, 17, 33, 1, 1, 64, 1, 1, 5, 1, 1, 1, 90, 1, 0]
    both(new, ctx, sum(new) + 3, 80, window=window, sinks=sinks)


@pytest.mark.parametrize("seqs,seed", [(255, 0), (256, 1), (257, 2), (1023, 3), (1024, 4), (1025, 5), (2300, 6)])
def test_many_requests_across_scans(seqs, seed):
    rng = random.Random(seed)
    new = [rng.choice([0, 1, 1, 1, rng.randint(2, 40)]) for _ in range(seqs)]
    ctx = [rng.choice([0, rng.randint(1, 300)]) for _ in range(seqs)]
    both(new, ctx, sum(new) + rng.randint(0, 9), rng.choice([22, 23, 37]), window=rng.choice([None, 48]), sinks=4)


def test_long_prompts_and_wide_tables():
    both([32768, 1, 5000], [0, 30000, 27768], 37769, 2048)
    both([1, 20000], [2**20, 12345], 20001, 65537)


def test_rows_that_do_not_fit_are_left_out():
    new, ctx = [3, 10, 1, 4], [20, 0, 50, 1]
    for rows in (0, 1, 3, 4, 12, 13, 14, 17):
        both(new, ctx, rows, 6)


def test_a_table_that_is_too_narrow_gives_its_rows_no_slot():
    both([40, 3], [0, 70], 43, 2)


def test_short_lists_negative_lengths_and_pages():
    new, ctx, rows = [20, -3, 5, 9], [-7, 40, -2**31, 28], 40
    pages = [3, -1, 9, 9, 2]  # entry 1 of the first request is not a page; the last request's are missing
    got = build_step_tables(i32(new), i32(ctx), i32(pages), rows, 3, pad_page=-5)
    check(got, formula(new, ctx, pages, rows, 3, pad_page=-5))
    check(build_step_tables(i32(new), i32(ctx), i32([]), rows, 3), formula(new, ctx, [], rows, 3))
    check(build_step_tables(i32([2**31 - 1]), i32([0]), i32([4]), 20, 2), StepTables(
        torch.tensor([[4, 0]], dtype=torch.int32), torch.tensor([0, 20], dtype=torch.int32),
        torch.tensor([2**31 - 1], dtype=torch.int32), torch.arange(20), torch.cat((torch.arange(64, 80), torch.full((4,), -1)))))


def test_strided_and_offset_lengths():
    new, ctx = [3, 1, 7], [5, 90, 0]
    wide = torch.full((3, 5), 77, dtype=torch.int32, device="cuda")
    wide[:, 1], wide[:, 3] = i32(new), i32(ctx)
    pages = list(range(20))
    listed = i32([99] + pages)[1:]
    check(build_step_tables(wide[:, 1], wide[:, 3], listed, 11, 6), formula(new, ctx, pages, 11, 6))


def test_on_another_stream_and_replayed():
    new, ctx, pages = i32([1] * 40), i32([0] * 40), i32(list(range(4000)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = build_step_tables(new, ctx, pages, 40, 9, window=32, sinks=1)
    side.synchronize()
    check(first, formula([1] * 40, [0] * 40, pages.tolist(), 40, 9, 32, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = build_step_tables(new, ctx, pages, 48, 9, window=32, sinks=1)
    rng = random.Random(0)
    for _ in range(4):
        lens = [rng.randint(0, 130) for _ in range(40)]
        rows = [rng.choice([0, 1, 1]) for _ in range(40)]
        new.copy_(i32(rows))
        ctx.copy_(i32(lens))
        graph.replay()
        torch.cuda.synchronize()
        check(got, formula(rows, lens, pages.tolist(), 48, 9, 32, 1))
        check(build_step_tables(new, ctx, pages, 48, 9, window=32, sinks=1), [t.cpu() for t in got])
