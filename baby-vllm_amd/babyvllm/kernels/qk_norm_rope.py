"""RMS norm of each query and key head, RoPE and KV-store append in one launch (no counterpart in the reference).

``fused_qk_norm_rope_and_cache`` is ``fused_rope_and_cache`` for models that normalise every
query and key head before the rotation: ``x · rsqrt(mean(x²) + eps) · weight`` over the head's
dimensions, then rotate-half RoPE, in fp32 and rounded once. q is returned in a new tensor (or
in ``out``); rotated k and raw v go to the cache rows of ``slot_mapping`` and nowhere else: the
inputs stay as they are. Slots outside the cache are not written; of two tokens with one slot,
either may be the one that stays.
"""

from __future__ import annotations

import torch

from babyvllm.kernels import _lib


def _range(t: torch.Tensor) -> tuple[int, int]:
    """First byte and the one behind the last that a non-empty tensor of positive strides spans."""
    span = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + span * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _range(a), _range(b)
    return a0 < b1 and b0 < a1


def fused_qk_norm_rope_and_cache(q, k, v, q_weight, k_weight, eps, cos, sin, kv_cache, slot_mapping, out=None):
    """Normalised, rotated q ``[T, H, D]``; k and v ``[T, Hkv, D]`` into the paged cache.

    ``q_weight`` and ``k_weight``: ``[D]`` vectors, both bf16 or both fp32. ``cos`` and ``sin``:
    ``[T, D]`` per-token rows (duplicated halves), both bf16 or both fp32. ``out``: where q
    goes: ``q`` itself, or a tensor that shares no memory with the others.
    """
    if out is None and q.is_cuda:
        got = _lib.fast().norm_rope(q, k, v, q_weight, k_weight, eps, cos, sin, kv_cache, slot_mapping, *_lib.current())
        if got is not None:
            return got
    for name, t in (("q", q), ("k", k), ("v", v), ("q_weight", q_weight), ("k_weight", k_weight), ("cos", cos),
                    ("sin", sin), ("kv_cache", kv_cache), ("slot_mapping", slot_mapping)):
        _lib.require_rocm_tensor(name, t)
        if t.device != q.device:
            raise RuntimeError(f"{name} is on {t.device}, q on {q.device}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3 or t.stride(-1) != 1:
            raise ValueError(f"{name} must be [T, heads, D] with a unit last stride, got shape {tuple(t.shape)}")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    num_tokens, num_heads, head_dim = q.shape
    num_kv_heads = k.shape[1]
    if k.shape[0] != num_tokens or k.shape[2] != head_dim or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match q {tuple(q.shape)}")
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    for names, (x, y), shape in ((("cos", "sin"), (cos, sin), None), (("q_weight", "k_weight"), (q_weight, k_weight), (head_dim,))):
        if x.dtype not in (torch.bfloat16, torch.float32) or y.dtype != x.dtype:
            raise TypeError(f"{names[0]} and {names[1]} must both be bfloat16 or both float32, got {x.dtype} and {y.dtype}")
        if shape is not None and (x.shape != shape or y.shape != shape or not x.is_contiguous() or not y.is_contiguous()):
            raise ValueError(f"{names[0]} and {names[1]} must be contiguous vectors of {head_dim}")
    if cos.dim() != 2 or cos.shape[0] < num_tokens or cos.shape[1] != head_dim or sin.shape != cos.shape \
            or cos.stride(1) != 1 or sin.stride(1) != 1:
        raise ValueError("cos/sin must be [num_tokens, head_dim] with a unit last stride")
    if kv_cache.dim() != 5 or kv_cache.shape[0] != 2 or kv_cache.shape[3] != num_kv_heads \
            or kv_cache.shape[4] != head_dim:
        raise ValueError(f"kv_cache must be [2, NB, BS, {num_kv_heads}, {head_dim}], got {tuple(kv_cache.shape)}")
    if kv_cache.dtype != torch.bfloat16:
        raise TypeError(f"kv_cache must be bfloat16, got {kv_cache.dtype}")
    if not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous (its [NB·BS, Hkv, D] view is written)")
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.shape[0] < num_tokens:
        raise TypeError("slot_mapping must be an int64 vector with one slot per token")
    if out is None:
        out = torch.empty(num_tokens, num_heads, head_dim, device=q.device, dtype=q.dtype)
    else:
        _lib.require_rocm_tensor("out", out)
        if out.device != q.device or out.dtype != q.dtype or out.shape != q.shape or out.stride(-1) != 1:
            raise ValueError("out must be a tensor of q's shape, type and device with a unit last stride")
        if any(n > 1 and step == 0 for n, step in zip(out.shape, out.stride())):
            raise ValueError("out's elements must not share memory")
        in_place = out.data_ptr() == q.data_ptr() and out.stride() == q.stride()
        others = (q_weight, k_weight, cos, sin, kv_cache, slot_mapping)
        if num_tokens and any(_overlap(out, t) for t in (others if in_place else (q, k, v) + others)):
            raise ValueError("out must be q itself or share no memory with the other tensors")
    if num_tokens == 0:
        return out
    slot_mapping = slot_mapping.contiguous()
    k_cache, v_cache = kv_cache[0], kv_cache[1]
    with torch.cuda.device(q.device):
        rc = _lib.lib().bvllm_qk_norm_rope_append(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
            v.data_ptr(), v.stride(0), v.stride(1),
            q_weight.data_ptr(), k_weight.data_ptr(), int(q_weight.dtype == torch.float32), float(eps),
            cos.data_ptr(), cos.stride(0), sin.data_ptr(), sin.stride(0), int(cos.dtype == torch.float32),
            out.data_ptr(), out.stride(0), out.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(1), k_cache.stride(2),
            kv_cache.shape[1] * kv_cache.shape[2], slot_mapping.data_ptr(),
            num_tokens, num_heads, num_kv_heads, head_dim, _lib.stream_handle(q.device))
    _lib.check(rc, "bvllm_qk_norm_rope_append")
    return out
