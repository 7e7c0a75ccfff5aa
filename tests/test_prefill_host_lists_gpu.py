"""Steps that leave rows of their requests out, with host lists of all rows: every row of the step is computed.

Bounds as in ``test_window_attn_gpu`` (a window of everything).
"""

import pytest
import torch

from babyvllm.kernels.paged_prefill import paged_prefill_attention
from babyvllm.kernels.step_tables import build_step_tables
from babyvllm.worker.context import AttentionMetadata
from tests._cases import python_path
from tests.test_window_attn_gpu import build, check, formula, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rows", [2, 5, 6, 8])
@pytest.mark.parametrize("ctx", [[150, 40, 300, 90], [6000, 40, 300, 900]], ids=str)
def test_host_lists_of_more_rows_than_the_step_has(ctx, rows, native, monkeypatch):
    if not native:
        python_path(monkeypatch)
    new = [5, 1, 1, 1]
    full, cache, whole = build(list(zip(ctx, new)), 2, 7, 64, 10**6, 0)
    held = [whole.block_tables[s, :-(-(c + n) // 16)] for s, (c, n) in enumerate(zip(ctx, new))]
    t = build_step_tables(i32(new), i32(ctx), torch.cat(held), rows, whole.block_tables.shape[1])
    md = AttentionMetadata(t.slot_mapping, t.block_tables, t.query_start_loc, t.seq_lens, i32(ctx), [0, 5, 6, 7, 8],
                           [c + n for c, n in zip(ctx, new)], ctx, 5, max(c + n for c, n in zip(ctx, new)))
    q = full[:rows].contiguous()
    spoilt = [torch.full_like(q, float("nan")) for _ in range(4)]  # what the output's memory held before
    torch.cuda.synchronize()
    del spoilt
    check(paged_prefill_attention(q, cache, md, 0.1), formula(q, cache, md, 0.1, 10**6, 0))
