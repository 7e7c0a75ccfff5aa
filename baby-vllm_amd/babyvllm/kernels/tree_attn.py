"""Attention of drafted token trees over the paged cache (no counterpart in the reference).

``paged_tree_attention(q, kv_cache, md, scale)`` is ``paged_prefill_attention``'s step
for speculative decoding: the rows of sequence s are its drafted tokens, a tree whose
node 0 is the last sampled token, with their K/V already appended behind the context
(node j at position ``context_lens[s] + j``, whatever its depth). A row attends the whole
context and the drafted tokens that its bits in ``md.tree_mask`` name:
int64 ``[T, W]``, bit ``j % 64`` of word ``j // 64`` for node j of the row's sequence, its
own bit among them. ``ancestor_masks`` makes the words (and the depths, which give the
rotary positions) from each node's parent.

A row that sees no key gives zeros, and a key that a row does not see does not reach it,
whatever it holds. Rows of ``q`` behind the last sequence are not computed. Long contexts
run in key ranges chosen from the step's host lists: the last bits of a row can depend on
the other sequences of the step. Scores, softmax statistics and sums are fp32. The weights of the
context's whole 64-key tiles are rounded to bf16 in ranges, as in ``paged_prefill_attention``; all
others, and all where the launch has no ranges, keep 16 bits. Ranges take fp32 scratch (at most
64 MiB); without the memory for it the launch that needs none runs.
"""

from __future__ import annotations

import torch

from babyvllm.kernels import _lib

_TILE = 64  # keys


def ancestor_masks(parents, words: int | None = None):
    """``(tree_mask, depths)`` of one step: CPU int64 ``[T, W]`` and ``[T]``.

    ``parents`` has one list per sequence: the parent node of each of its drafted tokens,
    -1 for a root (node 0, and any other node to start from the context alone); a parent
    comes before its children. Depth 0 is a root: node j's position is
    ``context_len + depths[j]``. ``words`` pads the masks to that many words.
    """
    need = -(-max((len(p) for p in parents), default=0) // 64)
    words = max(need, 1) if words is None else words
    if words < max(need, 1):
        raise ValueError(f"{words} words hold {64 * words} nodes, the largest tree has more")
    masks, depths = [], []
    for tree in parents:
        seen, depth = [], []
        for i, p in enumerate(tree):
            if not -1 <= p < i:
                raise ValueError(f"node {i} has parent {p}: parents come before their children")
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        for bits in seen:
            row = [bits >> 64 * w & (1 << 64) - 1 for w in range(words)]
            masks.append([v - (1 << 64) if v >> 63 else v for v in row])
        depths.extend(depth)
    return (torch.tensor(masks, dtype=torch.int64).view(len(masks), words),
            torch.tensor(depths, dtype=torch.int64))


def _key_tiles(md, num_seqs):
    """(64-key tiles of all sequences, of the longest) from the host list, -1 for each without it."""
    seq = getattr(md, "seq_lens_cpu", None)
    if seq is None or len(seq) != num_seqs:
        return -1, -1
    tiles = [(max(int(n), 0) + _TILE - 1) // _TILE for n in seq]
    return sum(tiles), max(tiles, default=0)


def paged_tree_attention(q, kv_cache, md, scale):
    """``[T, H, D]`` attention of drafted token trees, K/V read from the paged cache."""
    mask = getattr(md, "tree_mask", None)
    if mask is None:
        raise ValueError("md.tree_mask is missing: the drafted tokens' visibility words")
    if q.is_cuda:
        out = _lib.fast().tree(q, kv_cache, md.block_tables, md.query_start_loc, md.seq_lens, md.context_lens, mask,
                               getattr(md, "seq_lens_cpu", None), md.max_query_len, scale, *_lib.current())
        if out is not None:
            return out
    for name, t in (("q", q), ("kv_cache", kv_cache), ("block_tables", md.block_tables),
                    ("query_start_loc", md.query_start_loc), ("seq_lens", md.seq_lens),
                    ("context_lens", md.context_lens), ("tree_mask", mask)):
        _lib.require_rocm_tensor(name, t)
        if t.device != q.device:
            raise RuntimeError(f"{name} is on {t.device}, q on {q.device}")
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
    if mask.dtype != torch.int64:
        raise TypeError(f"tree_mask must be int64, got {mask.dtype}")
    num_tokens, num_heads, head_dim = q.shape
    _, num_blocks, page, num_kv_heads, cache_dim = kv_cache.shape
    if cache_dim != head_dim:
        raise ValueError("kv_cache head_dim differs from q")
    bt, max_query_len = md.block_tables, int(md.max_query_len)
    num_seqs = md.seq_lens.shape[0]
    if bt.dim() != 2 or bt.stride(1) != 1 or bt.shape[0] < num_seqs:
        raise ValueError("block_tables must be [S, W] with a unit last stride")
    if md.query_start_loc.shape != (num_seqs + 1,) or md.context_lens.shape != (num_seqs,):
        raise ValueError("query_start_loc must be [S + 1], seq_lens and context_lens [S]")
    if mask.dim() != 2 or mask.shape[0] < num_tokens or mask.stride(1) != 1 or mask.shape[1] * 64 < max_query_len:
        raise ValueError(f"tree_mask must be [T, W] with a unit last stride and a bit for each of {max_query_len} "
                         f"drafted tokens, got {tuple(mask.shape)}")
    k_cache, v_cache = kv_cache[0], kv_cache[1]
    if k_cache.stride(3) != 1:
        raise ValueError("K and V halves of kv_cache must have a unit last stride")

    out = torch.empty(num_tokens, num_heads, head_dim, device=q.device, dtype=q.dtype)
    if num_tokens == 0 or num_seqs == 0 or max_query_len == 0:
        return out
    qsl, seq_lens, ctx_lens = md.query_start_loc.contiguous(), md.seq_lens.contiguous(), md.context_lens.contiguous()
    h = _lib.lib()
    with torch.cuda.device(q.device):
        total, longest = _key_tiles(md, num_seqs)
        split = h.bvllm_tree_split_tiles(num_seqs, num_tokens, max_query_len, num_heads, num_kv_heads, head_dim,
                                         bt.shape[1], total, longest)
        ranges, workspace = 0, None
        if split != 0:
            ranges = h.bvllm_prefill_ranges(bt.shape[1], abs(split), longest)
            workspace = _lib.optional_scratch(h.bvllm_tree_workspace_bytes(num_tokens, num_heads, head_dim, ranges),
                                              q.device)
            if workspace is None:
                split = 0
        rc = h.bvllm_paged_tree_attention(
            q.data_ptr(), q.stride(0), q.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            num_blocks,
            bt.data_ptr(), bt.stride(0), bt.shape[1],
            qsl.data_ptr(), seq_lens.data_ptr(), ctx_lens.data_ptr(),
            mask.data_ptr(), mask.stride(0), mask.shape[1], float(scale),
            out.data_ptr(), out.stride(0), out.stride(1),
            num_seqs, num_tokens, max_query_len, num_heads, num_kv_heads, head_dim, page,
            None if workspace is None else workspace.data_ptr(), split, ranges, _lib.stream_handle(q.device))
    _lib.check(rc, "bvllm_paged_tree_attention")
    return out
