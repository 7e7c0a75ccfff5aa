"""Steps of single rows whose host lists say otherwise: the runs that their rows are cut into are added up all the same.

Bounds as in ``test_window_attn_gpu``.
"""

import ctypes

import pytest
import torch

from babyvllm.kernels import _lib
from babyvllm.kernels.step_tables import build_step_tables
from babyvllm.kernels.window_attn import paged_window_attention
from babyvllm.worker.context import AttentionMetadata
from tests._cases import python_path
from tests.test_window_attn_gpu import build, check, formula, i32, raw_call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("single", [-1, 0, 1, 3])
@pytest.mark.parametrize("heads", [(2, 7, 64), (1, 7, 128), (8, 1, 128)], ids=str)
def test_any_count_of_single_rows_gives_their_outputs(heads, single):
    q, cache, md = build([(2000, 1), (77, 1), (900, 1)], *heads, 1500, 20)
    want = formula(q, cache, md, 0.1, 1500, 20)
    for runs in (1, 2, 3, 16):
        print(runs, flush=True)
        check(raw_call(q, cache, md, 0.1, 1500, 20, 128, 0, runs, single), want)


@pytest.mark.parametrize("heads", [(2, 7, 64), (4, 7, 128)], ids=str)
def test_the_plan_of_a_step_of_single_rows_holds_for_a_count_of_none(heads):
    hkv, group, d = heads
    q, cache, md = build([(4000, 1)], *heads, 4096, 4)
    plan = (ctypes.c_int32 * 4)()
    assert _lib.lib().bvllm_window_plan(1, 1, 1, 0, hkv * group, hkv, d, md.block_tables.shape[1], 4096, 4, plan) == 0
    columns, split, _, runs = plan
    assert runs > 1
    check(raw_call(q, cache, md, 0.1, 4096, 4, columns, split, runs, 0), formula(q, cache, md, 0.1, 4096, 4))


@pytest.mark.parametrize("native", [True, False])
def test_a_request_of_which_the_step_has_one_row(native, monkeypatch):
    if not native:
        python_path(monkeypatch)
    # Five new tokens, a step of one row: the tables leave the others out, the host's lists do not.
    full, cache, whole = build([(3000, 5)], 4, 7, 128, 4096, 4)
    pages = whole.block_tables[0, :-(-3005 // 16)].contiguous()
    t = build_step_tables(i32([5]), i32([3000]), pages, 1, pages.shape[0])
    assert t.query_start_loc.tolist() == [0, 1]
    md = AttentionMetadata(t.slot_mapping, t.block_tables, t.query_start_loc, t.seq_lens, i32([3000]), [0, 5], [3005], [3000], 5, 3005)
    q = full[:1].contiguous()
    want = formula(q, cache, md, 0.1, 4096, 4)
    for _ in range(3):
        spoilt = [torch.full_like(q, float("nan")) for _ in range(4)]  # what the output's memory held before
        torch.cuda.synchronize()
        del spoilt
        check(paged_window_attention(q, cache, md, 0.1, 4096, 4), want)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rows", [1, 2, 5, 6])
def test_host_lists_of_more_rows_than_the_step_has(rows, native, monkeypatch):
    if not native:
        python_path(monkeypatch)
    # Requests of 5, 1, 1 and 1 new tokens, a step of fewer rows.
    new, ctx = [5, 1, 1, 1], [1500, 40, 300, 900]
    full, cache, whole = build(list(zip(ctx, new)), 2, 7, 64, 1000, 4)
    held = [whole.block_tables[s, :-(-(c + n) // 16)] for s, (c, n) in enumerate(zip(ctx, new))]
    t = build_step_tables(i32(new), i32(ctx), torch.cat(held), rows, whole.block_tables.shape[1])
    md = AttentionMetadata(t.slot_mapping, t.block_tables, t.query_start_loc, t.seq_lens, i32(ctx), [0, 5, 6, 7, 8],
                           [c + n for c, n in zip(ctx, new)], ctx, 5, 1505)
    q = full[:rows].contiguous()
    check(paged_window_attention(q, cache, md, 0.1, 1000, 4), formula(q, cache, md, 0.1, 1000, 4))
