"""Block tables and slot maps of a step from its requests' lengths (no counterpart in the reference).

``build_step_tables(query_lens, context_lens, pages, num_tokens, width)`` turns what a
scheduler knows of a step, every request's cached and new tokens and the pages it holds, into
the tensors that the cache and attention kernels take (``AttentionMetadata``), on the GPU and
without a look at the lengths on the host: one launch on the current stream, capturable.

* ``query_lens`` and ``context_lens``: int32 ``[S]``, new and cached tokens of each request
  (0 new ones for a row that is not in use); at most 2^20 requests.
* ``pages``: int32 ``[P]``, the requests' pages one request after another, each in the order of
  its positions: ``ceil((context + new) / 16)`` of them. With a ``window`` only those of its
  first ``sinks`` tokens and those from the page of position ``context - window + 1`` on: what
  ``paged_window_attention`` with the same ``window`` and ``sinks`` reads.
* ``num_tokens``: rows of the step. ``width``: entries of a table row.

Returns ``StepTables``: ``block_tables`` int32 ``[S, width]`` (``pad_page`` where a request
holds no page), ``query_start_loc`` int32 ``[S + 1]``, ``seq_lens`` int32 ``[S]``, ``positions``
and ``slot_mapping`` int64 ``[num_tokens]``. Rows behind the last request's have position 0 and
slot -1, which the append kernels do not write. Requests' rows beyond ``num_tokens`` are left
out (``query_start_loc`` ends there). A row whose page is not in the list, behind the table's
width or negative has slot -1; negative lengths count as 0.
"""

from __future__ import annotations

import operator
from typing import NamedTuple

import torch

from babyvllm.kernels import _lib

_MAX_WIDTH = 1 << 28  # of a sequence of 2^31 tokens and more
_MAX_SEQS = 1 << 20


class StepTables(NamedTuple):
    block_tables: torch.Tensor
    query_start_loc: torch.Tensor
    seq_lens: torch.Tensor
    positions: torch.Tensor
    slot_mapping: torch.Tensor


def build_step_tables(query_lens, context_lens, pages, num_tokens, width, *, window=None, sinks=0, pad_page=0):
    """The step's ``StepTables``. ``window`` None: the requests hold all their pages."""
    if query_lens.is_cuda:
        out = _lib.fast().tables(query_lens, context_lens, pages, num_tokens, width, window, sinks, pad_page, _MAX_WIDTH,
                                 *_lib.current())
        if out is not None:
            return StepTables._make(out)
    for name, t in (("query_lens", query_lens), ("context_lens", context_lens), ("pages", pages)):
        _lib.require_rocm_tensor(name, t)
        if t.device != query_lens.device:
            raise RuntimeError(f"{name} is on {t.device}, query_lens on {query_lens.device}")
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.dim() != 1:
            raise ValueError(f"{name} must be a vector, got shape {tuple(t.shape)}")
    num_seqs = query_lens.shape[0]
    if context_lens.shape[0] != num_seqs:
        raise ValueError(f"context_lens has {context_lens.shape[0]} requests, query_lens {num_seqs}")
    if num_seqs > _MAX_SEQS:
        raise ValueError(f"at most 2^20 requests, got {num_seqs}")
    num_tokens, width, sinks, pad_page = (operator.index(v) for v in (num_tokens, width, sinks, pad_page))
    window = None if window is None else operator.index(window)
    if not 0 <= num_tokens < 2**31 or not 1 <= width <= _MAX_WIDTH:
        raise ValueError(f"num_tokens must be from 0 to 2^31 - 1 and width from 1 to 2^28, got {num_tokens} and {width}")
    if not -2**31 <= pad_page < 2**31:
        raise ValueError(f"pad_page must fit 32 bits, got {pad_page}")
    if (window is not None and window < 1) or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    query_lens, context_lens, pages = query_lens.contiguous(), context_lens.contiguous(), pages.contiguous()
    device = query_lens.device
    out = StepTables(
        torch.empty(num_seqs, width, dtype=torch.int32, device=device),
        torch.empty(num_seqs + 1, dtype=torch.int32, device=device),
        torch.empty(num_seqs, dtype=torch.int32, device=device),
        torch.empty(num_tokens, dtype=torch.int64, device=device),
        torch.empty(num_tokens, dtype=torch.int64, device=device))
    with torch.cuda.device(device):
        rc = _lib.lib().bvllm_build_step_tables(
            query_lens.data_ptr(), context_lens.data_ptr(), num_seqs, pages.data_ptr(), pages.shape[0],
            0 if window is None else min(window, 2**31 - 1), min(sinks, 2**31 - 1), pad_page,
            out.block_tables.data_ptr(), width, out.query_start_loc.data_ptr(), out.seq_lens.data_ptr(),
            out.positions.data_ptr(), out.slot_mapping.data_ptr(), num_tokens, 16, _lib.stream_handle(device))
    _lib.check(rc, "bvllm_build_step_tables")
    return out
