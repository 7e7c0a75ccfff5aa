"""Draft trees and beams without a GPU: the trees' masks, and what the C entries and the wrappers refuse
(nothing is launched: the pointers below are never read)."""

import random

import pytest
import torch

from babyvllm.kernels import _lib
from babyvllm.kernels.tree_attn import ancestor_masks

P, BAD = 4096, 1


def test_masks_are_the_ancestors_and_depths_their_number():
    rng = random.Random(0)
    trees = [[-1], [], [-1, 0, 0, 1, 3], [-1, -1, 1, 0], [-1] + [rng.randrange(max(0, i - 3), i) for i in range(1, 150)]]
    mask, depth = ancestor_masks(trees)
    assert mask.dtype == torch.int64 and mask.shape == (160, 3) and depth.shape == (160,)
    row = 0
    for tree in trees:
        for i in range(len(tree)):
            line, p = {i}, tree[i]
            while p >= 0:
                line.add(p)
                p = tree[p]
            bits = [j for w in range(3) for j in range(64 * w, 64 * w + 64) if (int(mask[row, w]) >> (j - 64 * w)) & 1]
            assert set(bits) == line and depth[row] == len(line) - 1
            row += 1
    assert ancestor_masks([[-1, 0]], words=4)[0].shape == (2, 4)
    assert ancestor_masks([])[0].shape == (0, 1)


@pytest.mark.parametrize("tree", [[0], [-1, 1], [-1, 2, 0], [-2], [-1, 0, 5]])
def test_parents_behind_their_children_are_refused(tree):
    with pytest.raises(ValueError, match="parents come before"):
        ancestor_masks([tree])


def test_too_few_words_are_refused():
    with pytest.raises(ValueError, match="words"):
        ancestor_masks([list(range(-1, 64))], words=1)


def tree(**k):
    a = dict(q=P, q_st=1792, q_sh=128, k=P, v=P, sb=8192, st=512, sh=128, nb=10, bt=P, bts=8, mb=8, qsl=P, seq=P, ctx=P,
             mask=P, ms=1, mw=1, scale=0.1, out=P, o_st=1792, o_sh=128, s=2, t=0, mq=8, h=14, hkv=2, d=128, bs=16, ws=P,
             split=0, ranges=0, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_paged_tree_attention(*{**a, **k}.values())


def test_tree_attention_refuses_on_the_host():
    assert tree() == 0 and tree(t=5, s=0) == 0 and tree(t=5, mq=0) == 0  # nothing to do
    bad = [dict(h=15), dict(d=96), dict(bs=32), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
           dict(scale=float("inf")), dict(t=-1), dict(s=-1), dict(hkv=0)]
    assert [k for k in bad if tree(**k) != BAD] == []
    bad = [dict(q=None), dict(mask=None), dict(k=None), dict(qsl=None), dict(q=P + 2), dict(q_st=1790), dict(sb=0), dict(sb=8190),
           dict(nb=0), dict(mb=0), dict(bts=7), dict(mw=0), dict(mq=65), dict(ms=0), dict(split=-1), dict(split=1 << 21), dict(split=-1 << 21, ranges=1), dict(split=-1, ranges=3),
           dict(split=1, ranges=0), dict(split=1, ranges=3), dict(split=1, ranges=2, ws=None),
           dict(split=1, ranges=2, ws=P + 4), dict(t=1 << 28), dict(st=1 << 28)]
    assert [k for k in bad if tree(**{"t": 16, **k}) != BAD] == []


def test_context_ranges_fit_the_table_and_the_scratch():
    h = _lib.lib()
    rng = random.Random(0)
    taken = [0, 0]
    for _ in range(2000):
        seqs, n = rng.randint(1, 70), rng.randint(1, 200)
        heads, hkv, d = rng.choice([(28, 4, 128), (14, 2, 64), (8, 8, 64), (20, 1, 128)])
        width = rng.choice([1, 2, 7, 130, 2049, 100000])
        known = rng.random() < 0.7
        longest = rng.randint(0, (width + 3) // 4 + 3) if known else -1
        total = rng.randint(longest, max(longest, longest * seqs)) if known else -1
        split = h.bvllm_tree_split_tiles(seqs, seqs * n, n, heads, hkv, d, width, total, longest)
        if split:
            taken[split > 0] += 1
            ranges = h.bvllm_prefill_ranges(width, abs(split), longest)
            assert 1 <= ranges <= h.bvllm_prefill_ranges(width, abs(split), -1)
            assert h.bvllm_tree_workspace_bytes(seqs * n, heads, d, ranges) == (ranges + 1) * seqs * n * heads * (d + 2) * 4 <= 64 << 20
    assert min(taken) > 200
    assert h.bvllm_tree_workspace_bytes(8, 28, 128, 0) == 0
    # One short chat stays on one launch; a long document does not.
    assert h.bvllm_tree_split_tiles(1, 8, 8, 14, 2, 64, 20, 5, 5) == 0
    assert h.bvllm_tree_split_tiles(1, 25, 25, 28, 4, 128, 2002, 501, 501) < 0
    assert h.bvllm_tree_split_tiles(16, 1024, 64, 28, 4, 128, 504, 900, 126) > 0


def layers(*pointers):
    import ctypes
    return (ctypes.c_void_p * len(pointers))(*pointers)


def commit(**k):
    a = dict(k=layers(P, 2 * P), v=layers(P, P), n=2, sb=8192, st=512, sh=128, nb=10, hkv=4, d=128, bs=16, bt=P, bts=8, mb=8,
             qsl=P, ctx=P, draft=P, target=P, parents=P, path=P, acc=P, fol=P, s=0, mp=8, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_commit_draft_tree(*{**a, **k}.values())


def test_commit_refuses_on_the_host():
    assert commit() == 0 and commit(n=0, k=None, v=None) == 0
    bad = [dict(n=-1), dict(n=2, k=None), dict(k=layers(P, None)), dict(k=layers(P, P)), dict(v=layers(P, P + 2)), dict(bs=8), dict(d=12), dict(hkv=0),
           dict(mp=0), dict(mp=4097), dict(s=-1), dict(s=65536), dict(sb=0), dict(hkv=1 << 18)]
    assert [k for k in bad if commit(**k) != BAD] == []
    bad = [dict(bt=None), dict(mb=0), dict(bts=7), dict(qsl=None), dict(ctx=None), dict(draft=None), dict(target=None),
           dict(parents=None), dict(path=None), dict(acc=None), dict(fol=None)]
    assert [k for k in bad if commit(**{"s": 1, **k}) != BAD] == []


def select(**k):
    a = dict(x=P, st=1000, fp32=0, scores=P, g=0, k=4, v=1000, n=8, ws=P, os=P, ob=P, ot=P, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_beam_select(*{**a, **k}.values())


def test_select_refuses_on_the_host():
    assert select() == 0
    bad = [dict(g=-1), dict(k=0), dict(k=33), dict(v=0), dict(n=0), dict(n=65), dict(v=1, n=5), dict(fp32=2),
           dict(k=32, v=524289)]
    assert [k for k in bad if select(**k) != BAD] == []
    assert select(k=32, v=524288, st=524288) == 0
    bad = [dict(x=None), dict(scores=None), dict(ws=None), dict(os=None), dict(ob=None), dict(ot=None), dict(st=-1),
           dict(ws=P + 4), dict(x=P + 1), dict(x=P + 2, fp32=1)]
    assert [k for k in bad if select(**{"g": 1, **k}) != BAD] == []
    assert _lib.lib().bvllm_beam_workspace_bytes(8, 2049) == 8 * 2 * 8


def reorder(**k):
    a = dict(k=layers(P), v=layers(P), n=1, sb=8192, st=512, sh=128, nb=10, hkv=4, d=128, bs=16, bt=P, bts=8, mb=8, seq=P,
             beams=P, g=0, kk=4, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_reorder_beams(*{**a, **k}.values())


def test_reorder_refuses_on_the_host():
    assert reorder() == 0
    bad = [dict(g=-1), dict(g=65536), dict(kk=0), dict(kk=33), dict(k=layers(None)), dict(bs=32), dict(st=4)]
    assert [k for k in bad if reorder(**k) != BAD] == []
    bad = [dict(bt=None), dict(bts=7), dict(mb=0), dict(seq=None), dict(beams=None)]
    assert [k for k in bad if reorder(**{"g": 1, **k}) != BAD] == []


def test_wrappers_refuse_cpu_tensors():
    from types import SimpleNamespace

    from babyvllm.kernels.beam import beam_select, reorder_beams
    from babyvllm.kernels.tree_attn import paged_tree_attention
    from babyvllm.kernels.tree_commit import commit_draft_tree

    i32 = torch.zeros(2, dtype=torch.int32)
    md = SimpleNamespace(block_tables=i32[None], query_start_loc=i32, seq_lens=i32[:1], context_lens=i32[:1],
                         max_query_len=1, tree_mask=torch.ones(1, 1, dtype=torch.int64))
    q, cache = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 16, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: paged_tree_attention(q, cache, md, 0.1),
                 lambda: commit_draft_tree([cache], md, i32[:1].long(), i32[:1].long(), i32[:1]),
                 lambda: beam_select(torch.zeros(2, 8), torch.zeros(2), 2),
                 lambda: reorder_beams([cache], i32[:, None], i32, torch.zeros(1, 2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()
