"""The list of a step's pages that the runner sends to the GPU, and what it refuses."""

import pytest

from babyvllm.sequence import SamplingParams, Sequence
from babyvllm.worker.model_runner import listed_pages


def requests(n):
    return [Sequence([5], SamplingParams(temperature=0.0)) for _ in range(n)]


@pytest.mark.parametrize("lengths,tables,bad", [
    ([17, 16], [[1], [2]], 0), ([16, 17], [[1], [2]], 1), ([16, 33, 1], [[1], [2, 3], [4]], 1), ([16, 1], [[1], []], 1),
])
def test_a_table_that_ends_before_its_request_is_refused(lengths, tables, bad):
    seqs = requests(len(lengths))
    with pytest.raises(ValueError, match=f"request {seqs[bad].seq_id} "):
        listed_pages(seqs, tables, lengths, 16)


@pytest.mark.parametrize("lengths,tables,want", [
    ([16, 17], [[1], [2, 3]], [1, 2, 3]), ([16, 17], [[1, 6, 7], [2, 3]], [1, 2, 3]), ([1, 0, 31], [[9, 8], [], [4, 5]], [9, 4, 5]),
    ([0], [[3]], []),
])
def test_each_request_has_as_many_pages_as_its_tokens_take(lengths, tables, want):
    kept = [list(t) for t in tables]
    assert listed_pages(requests(len(lengths)), tables, lengths, 16) == want and tables == kept
