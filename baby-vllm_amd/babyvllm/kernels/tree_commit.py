"""Taking over a verified draft tree (no counterpart in the reference).

After a step whose rows were drafted token trees (``paged_tree_attention``), the model's
answer at every node is known (``greedy_argmax`` of the logits, or a sampled token).
``commit_draft_tree(kv_caches, md, draft_tokens, target_tokens, parents)`` walks each
sequence's tree from node 0, always to the first child whose drafted token is the answer
at the node, and moves the K/V rows of the path, in every layer, to the positions right
behind the context, where the next step expects them. It returns, on the device and without
a host sync, ``(path, accepted, following)``: int32 ``[S, max_path]`` node numbers (-1 behind
the path), int32 ``[S]`` their count (the tokens that are in the cache now, node 0 among
them) and int64 ``[S]`` the answer at the path's end, the next step's node 0.
"""

from __future__ import annotations

import ctypes

import torch

from babyvllm.kernels import _lib

MAX_PATH = 4096


def layer_caches(kv_caches, device):
    """(layers, their pointer arrays, one of them) after checking that all have one shape and layout."""
    caches = list(kv_caches)
    for i, c in enumerate(caches):
        _lib.require_rocm_tensor(f"kv_caches[{i}]", c)
        if c.device != device:
            raise RuntimeError(f"kv_caches[{i}] is on {c.device}, not on {device}")
        if c.dtype != torch.bfloat16:
            raise TypeError(f"kv_caches[{i}] must be bfloat16, got {c.dtype}")
        if c.dim() != 5 or c.shape[0] != 2 or c.stride(4) != 1:
            raise ValueError(f"kv_caches[{i}] must be [2, NB, BS, Hkv, D] with a unit last stride, got {tuple(c.shape)}")
        if c.shape != caches[0].shape or c.stride() != caches[0].stride():
            raise ValueError(f"kv_caches[{i}] has another shape or layout than kv_caches[0]")
    if len({c.data_ptr() for c in caches}) < len(caches):
        raise ValueError("a cache is in kv_caches twice")
    k = (ctypes.c_void_p * max(1, len(caches)))(*[c.data_ptr() for c in caches])
    v = (ctypes.c_void_p * max(1, len(caches)))(*[c[1].data_ptr() for c in caches])
    return caches, k, v


def cache_shape(caches):
    """The C call's stride, page and head arguments (any valid ones without layers)."""
    if not caches:
        return 16 * 8, 8, 8, 1, 1, 8, 16
    _, num_blocks, page, hkv, d = caches[0].shape
    return (*caches[0].stride()[1:4], num_blocks, hkv, d, page)


def commit_draft_tree(kv_caches, md, draft_tokens, target_tokens, parents, max_path: int | None = None):
    """Moves the verified paths' K/V behind the contexts; returns ``(path, accepted, following)``.

    ``kv_caches`` are the layers' caches (all of one shape, each once; none: only the walk).
    ``draft_tokens`` and ``target_tokens`` int64 ``[T]`` and ``parents`` int32 ``[T]`` (node
    numbers within the sequence, before their children; -1 for the root) follow ``md.query_start_loc``.
    ``max_path`` bounds the accepted nodes (default ``md.max_query_len``, at most 4096).
    """
    bt, qsl, ctx = md.block_tables, md.query_start_loc, md.context_lens
    max_path = min(max(1, md.max_query_len), MAX_PATH) if max_path is None else max_path
    if draft_tokens.is_cuda:
        done = _lib.fast().commit(kv_caches, bt, qsl, ctx, draft_tokens, target_tokens, parents, max_path,
                                  *_lib.current())
        if done is not None:
            return done
    device = draft_tokens.device
    for name, t in (("draft_tokens", draft_tokens), ("target_tokens", target_tokens), ("parents", parents),
                    ("block_tables", bt), ("query_start_loc", qsl), ("context_lens", ctx)):
        _lib.require_rocm_tensor(name, t)
        if t.device != device:
            raise RuntimeError(f"{name} is on {t.device}, draft_tokens on {device}")
        want = torch.int64 if name.endswith("_tokens") else torch.int32
        if t.dtype != want:
            raise TypeError(f"{name} must be {want}, got {t.dtype}")
    for name, t in (("draft_tokens", draft_tokens), ("target_tokens", target_tokens), ("parents", parents)):
        if t.dim() != 1 or t.shape != draft_tokens.shape:
            raise ValueError("draft_tokens, target_tokens and parents must be vectors of one length")
    num_seqs = ctx.shape[0]
    if qsl.shape != (num_seqs + 1,) or ctx.dim() != 1:
        raise ValueError("query_start_loc must be [S + 1], context_lens [S]")
    if bt.dim() != 2 or bt.stride(1) != 1 or bt.shape[0] < num_seqs:
        raise ValueError("block_tables must be [S, W] with a unit last stride")
    max_path = int(max_path)
    if not 1 <= max_path <= MAX_PATH:
        raise ValueError(f"max_path must be 1 to {MAX_PATH}, got {max_path}")
    caches, k, v = layer_caches(kv_caches, device)
    path = torch.empty(num_seqs, max_path, device=device, dtype=torch.int32)
    accepted = torch.empty(num_seqs, device=device, dtype=torch.int32)
    following = torch.empty(num_seqs, device=device, dtype=torch.int64)
    if num_seqs == 0:
        return path, accepted, following
    if bt.shape[1] == 0 or draft_tokens.shape[0] == 0:
        raise ValueError("a commit needs drafted tokens and a block table")
    draft, target, par = draft_tokens.contiguous(), target_tokens.contiguous(), parents.contiguous()
    qsl, ctx = qsl.contiguous(), ctx.contiguous()
    with torch.cuda.device(device):
        rc = _lib.lib().bvllm_commit_draft_tree(
            k, v, len(caches), *cache_shape(caches), bt.data_ptr(), bt.stride(0), bt.shape[1],
            qsl.data_ptr(), ctx.data_ptr(), draft.data_ptr(), target.data_ptr(), par.data_ptr(),
            path.data_ptr(), accepted.data_ptr(), following.data_ptr(), num_seqs, max_path,
            _lib.stream_handle(device))
    _lib.check(rc, "bvllm_commit_draft_tree")
    return path, accepted, following
