"""What the runner makes of a scheduler's step on the GPU: its lists, as they were given."""

import pytest
import torch

from babyvllm.sequence import SamplingParams, Sequence
from tests.test_windowed_model_gpu import config

pytestmark = pytest.mark.gpu
PAGE = 16


def runner_of(blocks=24):
    from babyvllm.config import CacheConfig
    from babyvllm.worker.model_runner import ModelRunner
    runner = ModelRunner(config(), cache_config=CacheConfig(num_gpu_blocks=blocks), seed=3, init_std=0.1)
    runner.allocate_kv_cache()
    return runner


def step_of(specs, tables, slots=None):
    """(cached, new) tokens of each request; its pages' slots where none are given."""
    from babyvllm.scheduler import SchedulerOutput
    seqs, n, t, m = [], {}, {}, {}
    for i, ((ctx, new), table) in enumerate(zip(specs, tables)):
        seq = Sequence([(7 * i + 3 * j) % 500 for j in range(ctx + new)], SamplingParams(temperature=0.0))
        seq.num_computed_tokens = ctx
        seqs.append(seq)
        n[seq.seq_id], t[seq.seq_id] = new, table
        m[seq.seq_id] = slots[i] if slots else [table[p // PAGE] * PAGE + p % PAGE for p in range(ctx, ctx + new)]
    return SchedulerOutput(seqs, n, t, m, [])


SPECS = [(0, 20), (33, 1), (15, 9)]
TABLES = [[4, 9], [1, 7, 3, 11], [8, 2]]


def test_a_step_from_the_tables():
    runner = runner_of()
    out = step_of(SPECS, TABLES)
    ids, positions, md = runner.prepare_inputs(out)
    assert ids.tolist() == [t for s in out.scheduled_sequences for t in s.token_ids[s.num_computed_tokens:]]
    assert positions.tolist() == [p for c, n in SPECS for p in range(c, c + n)]
    assert md.slot_mapping.tolist() == [x for s in out.scheduled_sequences for x in out.slot_mappings[s.seq_id]]
    assert [t.dtype for t in (ids, positions, md.slot_mapping)] == [torch.int64] * 3
    assert md.block_tables.tolist() == [[4, 9, 0, 0], [1, 7, 3, 0], [8, 2, 0, 0]]
    assert md.query_start_loc.tolist() == [0, 20, 21, 30] and md.seq_lens.tolist() == [20, 34, 24]
    assert md.context_lens.tolist() == [0, 33, 15]


def test_the_schedulers_slots_are_the_steps():
    # Tokens that are not to be stored, and one that goes to a page outside its request's table.
    runner = runner_of()
    slots = [[4 * PAGE + p for p in range(16)] + [-1, -1, 9 * PAGE + 2, 9 * PAGE + 3], [5 * PAGE + 6], [-1] * 9]
    out = step_of(SPECS, TABLES, slots)
    _, _, md = runner.prepare_inputs(out)
    given = sum(slots, [])
    assert md.slot_mapping.tolist() == given
    for layer in runner._attention_layers():
        layer.kv_cache.fill_(3.0)
    runner.execute_model(out)
    for layer in runner._attention_layers():
        rows = layer.kv_cache.view(2, -1, *layer.kv_cache.shape[3:])
        written = (rows != 3.0).flatten(2).any(-1)  # [2, slots]
        for half in written:
            assert half.nonzero().flatten().tolist() == sorted(x for x in given if x >= 0)


@pytest.mark.parametrize("short", [0, 1, 2])
def test_a_table_that_ends_before_its_request_is_refused(short):
    # Its neighbours' pages would be taken for its own, and theirs for the next requests'.
    runner = runner_of()
    out = step_of(SPECS, TABLES)
    seq = out.scheduled_sequences[short].seq_id
    out.block_tables[seq] = out.block_tables[seq][:-1] if short != 1 else out.block_tables[seq][:2]
    with pytest.raises(ValueError, match=f"request {seq} "):
        runner.prepare_inputs(out)
