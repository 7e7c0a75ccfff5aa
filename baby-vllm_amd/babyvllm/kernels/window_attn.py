"""Attention of a sliding window and a few first tokens over the paged cache (no counterpart in the reference).

``paged_window_attention(q, kv_cache, md, scale, window, sinks=0)`` is the attention of a layer
whose rows see their last ``window`` keys, their own among them, and the sequence's first
``sinks`` tokens: the row at position p sees key j where ``j <= p`` and ``j > p - window`` or
``j < sinks`` (and ``j < seq_lens[s]``, inside the table). It takes a step's metadata as
``paged_prefill_attention`` does: decode steps, prompts behind cached tokens, and both at once,
the rows of sequence s at positions ``context_lens[s]`` and on, their K/V already in the cache.

Pages that no row of a sequence sees are not read for a result: their table entries may name any
page (``build_step_tables`` with the same ``window`` and ``sinks`` leaves them out), so that a
cache can give them back. A row that sees no key gives zeros, and a key that a row does not see
does not reach it, whatever it holds. Rows of ``q`` behind the last sequence are not computed.

``md.max_query_len`` bounds the query rows of every sequence. Few rows behind long windows are cut over more
work-groups, chosen from host sizes and (outside a capture) the list ``md.query_start_loc_cpu``: the last bits of a row can
depend on the other sequences of the step. That takes fp32 scratch (at most 128 MiB); without the memory
for it the launch that needs none runs. Scores, softmax statistics and sums are fp32. The weights of sequences of one row keep
16 bits, those of several rows are rounded to bf16, as in ``paged_prefill_attention``.
"""

from __future__ import annotations

import ctypes
import operator

import torch

from babyvllm.kernels import _lib
from babyvllm.kernels.paged_prefill import _single_query_seqs

_MAX = 2**31 - 1


def paged_window_attention(q, kv_cache, md, scale, window, sinks=0):
    """``[T, H, D]`` attention of the step's rows, K/V read from the paged cache."""
    # (A captured step is replayed with other sequences than its host lists': they do not steer it.)
    host_lists = not (q.is_cuda and torch._C._cuda_isCurrentStreamCapturing())
    if q.is_cuda:
        out = _lib.fast().window(q, kv_cache, md.block_tables, md.query_start_loc, md.seq_lens, md.context_lens,
                                 getattr(md, "query_start_loc_cpu", None) if host_lists else None, md.max_query_len,
                                 scale, window, sinks, *_lib.current())
        if out is not None:
            return out
    for name, t in (("q", q), ("kv_cache", kv_cache), ("block_tables", md.block_tables),
                    ("query_start_loc", md.query_start_loc), ("seq_lens", md.seq_lens),
                    ("context_lens", md.context_lens)):
        _lib.require_rocm_tensor(name, t)
        if t.device != q.device:
            raise RuntimeError(f"{name} is on {t.device}, q on {q.device}")
    window, sinks = min(operator.index(window), _MAX), min(operator.index(sinks), _MAX)
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    if q.dim() != 3 or q.stride(-1) != 1:
        raise ValueError("q must be [T, H, D] with a unit last stride")
    if q.dtype != torch.bfloat16 or kv_cache.dtype != torch.bfloat16:
        raise TypeError("q and kv_cache must be bfloat16")
    if kv_cache.dim() != 5 or kv_cache.shape[0] != 2:
        raise ValueError(f"kv_cache must be [2, NB, BS, Hkv, D], got {tuple(kv_cache.shape)}")
    for name, t in (("block_tables", md.block_tables), ("query_start_loc", md.query_start_loc),
                    ("seq_lens", md.seq_lens), ("context_lens", md.context_lens)):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
    num_tokens, num_heads, head_dim = q.shape
    _, num_blocks, page, num_kv_heads, cache_dim = kv_cache.shape
    if cache_dim != head_dim:
        raise ValueError("kv_cache head_dim differs from q")
    bt, max_query_len = md.block_tables, int(md.max_query_len)
    if md.seq_lens.dim() != 1:
        raise ValueError("seq_lens must be [S]")
    num_seqs = md.seq_lens.shape[0]
    if bt.dim() != 2 or bt.stride(1) != 1 or bt.shape[0] < num_seqs:
        raise ValueError("block_tables must be [S, W] with a unit last stride")
    if md.query_start_loc.shape != (num_seqs + 1,) or md.context_lens.shape != (num_seqs,):
        raise ValueError("query_start_loc must be [S + 1], seq_lens and context_lens [S]")
    k_cache, v_cache = kv_cache[0], kv_cache[1]
    if k_cache.stride(3) != 1:
        raise ValueError("K and V halves of kv_cache must have a unit last stride")

    out = torch.empty(num_tokens, num_heads, head_dim, device=q.device, dtype=q.dtype)
    if num_tokens == 0 or num_seqs == 0 or max_query_len == 0:
        return out
    qsl, seq_lens, ctx_lens = md.query_start_loc.contiguous(), md.seq_lens.contiguous(), md.context_lens.contiguous()
    h = _lib.lib()
    single = _single_query_seqs(md, num_seqs) if max_query_len > 1 and host_lists else -1
    if single >= 0 and md.query_start_loc_cpu[-1] > num_tokens:
        single = -1  # another step's list: this one leaves rows out
    with torch.cuda.device(q.device):
        plan = (ctypes.c_int32 * 4)()
        _lib.check(h.bvllm_window_plan(num_seqs, num_tokens, max_query_len, single, num_heads, num_kv_heads, head_dim,
                                       bt.shape[1], window, sinks, plan), "bvllm_window_plan")
        columns, split_tiles, num_ranges, row_runs = plan
        nbytes = h.bvllm_window_workspace_bytes(num_seqs, num_tokens, num_heads, head_dim, num_ranges, row_runs)
        workspace = _lib.optional_scratch(nbytes, q.device) if nbytes > 0 else None
        if workspace is None:
            split_tiles, num_ranges, row_runs = 0, 0, 1
        rc = h.bvllm_paged_window_attention(
            q.data_ptr(), q.stride(0), q.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            num_blocks,
            bt.data_ptr(), bt.stride(0), bt.shape[1],
            qsl.data_ptr(), seq_lens.data_ptr(), ctx_lens.data_ptr(),
            window, sinks, float(scale),
            out.data_ptr(), out.stride(0), out.stride(1),
            num_seqs, num_tokens, max_query_len, single,
            num_heads, num_kv_heads, head_dim, page, None if workspace is None else workspace.data_ptr(),
            columns, split_tiles, num_ranges, row_runs, _lib.stream_handle(q.device))
    _lib.check(rc, "bvllm_paged_window_attention")
    return out
