"""Beam search over the paged cache (no counterpart in the reference).

``beam_select(logits, scores, num_beams)`` picks each group's best continuations from its
beams' logits, as ``greedy_argmax`` does for one candidate;
``reorder_beams(kv_caches, block_tables, seq_lens, beams)`` then gives every surviving beam
its parent's context: full pages are shared through the block tables, the page being
filled is copied. Neither syncs with the host, so both can sit in a captured decode graph.
"""

from __future__ import annotations

import torch

from babyvllm.kernels import _lib
from babyvllm.kernels.tree_commit import cache_shape, layer_caches

MAX_BEAMS = 32
MAX_CANDIDATES = 64


def beam_select(logits, scores, num_beams: int, num_candidates: int | None = None):
    """The best continuations of every group of ``num_beams`` rows: ``(scores, beams, tokens)``.

    ``logits`` ``[G * K, vocab]`` bf16 or fp32 with unit column stride (rows may be one, expanded), ``scores`` fp32 (one
    per row, in any shape): the beams' summed log-probabilities. A continuation's total is
    ``score + logit - logsumexp(logits of the beam)``. Returned are the ``num_candidates``
    (default ``2 * K``, at most 64) best of each group, fp32 totals, int64 beam numbers within
    the group and int64 tokens, each ``[G, num_candidates]``, in descending order, equal totals
    by ``beam * vocab + token``. Totals are added up and compared in 64 bits, but a row's logsumexp
    is a sum of 32-bit exponentials, off by less than 2^-17 (3e-7 as measured): a beam's
    tokens are in the order of their logits, and beams of equal logits and scores have equal
    totals, while totals of different beams that are closer than that can come in either
    order. A beam whose score is not finite (an unused one: -inf), or whose logits hold a NaN,
    a +inf or no finite value, has totals of -inf.
    """
    if num_candidates is None and logits.dim() == 2:
        num_candidates = min(2 * num_beams, num_beams * logits.shape[1])
    if logits.is_cuda:
        done = _lib.fast().beam(logits, scores, num_beams, num_candidates, MAX_BEAMS, MAX_CANDIDATES, *_lib.current())
        if done is not None:
            return done
    _lib.require_rocm_tensor("logits", logits)
    _lib.require_rocm_tensor("scores", scores)
    if scores.device != logits.device:
        raise RuntimeError(f"scores are on {scores.device}, logits on {logits.device}")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be [G * K, vocab] with a unit column stride")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    if scores.dtype != torch.float32:
        raise TypeError(f"scores must be float32, got {scores.dtype}")
    rows, vocab = logits.shape
    if not 1 <= num_beams <= MAX_BEAMS or rows % num_beams:
        raise ValueError(f"num_beams must be 1 to {MAX_BEAMS} and divide the {rows} rows, got {num_beams}")
    if scores.numel() != rows:
        raise ValueError(f"scores has {scores.numel()} values for {rows} rows")
    n = int(num_candidates)
    if not 1 <= n <= min(MAX_CANDIDATES, num_beams * vocab):
        raise ValueError(f"num_candidates must be 1 to {min(MAX_CANDIDATES, num_beams * vocab)}, got {n}")
    groups = rows // num_beams
    out_scores = torch.empty(groups, n, device=logits.device, dtype=torch.float32)
    out_beams = torch.empty(groups, n, device=logits.device, dtype=torch.int64)
    out_tokens = torch.empty_like(out_beams)
    if groups == 0:
        return out_scores, out_beams, out_tokens
    scores = scores.contiguous()
    h = _lib.lib()
    with torch.cuda.device(logits.device):
        ws = torch.empty(h.bvllm_beam_workspace_bytes(rows, vocab) // 4, device=logits.device, dtype=torch.float32)
        rc = h.bvllm_beam_select(logits.data_ptr(), logits.stride(0) if rows > 1 else vocab,
                                 1 if logits.dtype == torch.float32 else 0, scores.data_ptr(), groups, num_beams,
                                 vocab, n, ws.data_ptr(), out_scores.data_ptr(), out_beams.data_ptr(),
                                 out_tokens.data_ptr(), _lib.stream_handle(logits.device))
    _lib.check(rc, "bvllm_beam_select")
    return out_scores, out_beams, out_tokens


def reorder_beams(kv_caches, block_tables, seq_lens, beams):
    """Gives beam b of every group the context of beam ``beams[g, b]`` of it, in place; returns the tables.

    ``block_tables`` int32 ``[G * K, W]``, ``seq_lens`` int32 ``[G * K]`` (the tokens in the
    cache; equal within a group, whose first row counts), ``beams`` int64 ``[G, K]`` (an index
    outside the group leaves its beam as it is). The entries of the ``seq_len // 16`` full
    pages are taken from the parent's row; the entry behind them, the page being filled, must
    be the beam's own page: it stays, and its ``seq_len % 16`` tokens are copied from the
    parent's page in every layer of ``kv_caches``. A parent may be named any number of times,
    and by beams that are parents themselves: everything is read before it is overwritten.
    Nothing is copied from or to a page outside the pool.
    """
    if block_tables.is_cuda:
        if _lib.fast().reorder(kv_caches, block_tables, seq_lens, beams, MAX_BEAMS, *_lib.current()):
            return block_tables
    for name, t, dtype in (("block_tables", block_tables, torch.int32), ("seq_lens", seq_lens, torch.int32),
                           ("beams", beams, torch.int64)):
        _lib.require_rocm_tensor(name, t)
        if t.device != block_tables.device:
            raise RuntimeError(f"{name} is on {t.device}, block_tables on {block_tables.device}")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if beams.dim() != 2 or beams.shape[1] > MAX_BEAMS:
        raise ValueError(f"beams must be [G, K] with K at most {MAX_BEAMS}, got {tuple(beams.shape)}")
    groups, k = beams.shape
    if block_tables.dim() != 2 or block_tables.shape[0] != groups * k or block_tables.stride(1) != 1:
        raise ValueError(f"block_tables must be [{groups * k}, W] with a unit last stride, got {tuple(block_tables.shape)}")
    if groups * k > 1 and block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError("block_tables must not overlap: every row is written")
    if seq_lens.shape != (groups * k,):
        raise ValueError(f"seq_lens must be [{groups * k}], got {tuple(seq_lens.shape)}")
    caches, kp, vp = layer_caches(kv_caches, block_tables.device)
    if groups * k == 0 or block_tables.shape[1] == 0:
        return block_tables
    lens, parents = seq_lens.contiguous(), beams.contiguous()
    width = block_tables.shape[1]
    with torch.cuda.device(block_tables.device):
        rc = _lib.lib().bvllm_reorder_beams(
            kp, vp, len(caches), *cache_shape(caches), block_tables.data_ptr(), block_tables.stride(0) if groups * k > 1 else width,
            width, lens.data_ptr(), parents.data_ptr(), groups, k, _lib.stream_handle(block_tables.device))
    _lib.check(rc, "bvllm_reorder_beams")
    return block_tables
