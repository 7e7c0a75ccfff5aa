"""The calls of a windowed step without a GPU: what the C entries and the wrappers refuse (nothing is
launched: the pointers below are never read)."""

import ctypes
import random

import pytest
import torch

from babyvllm.kernels import _lib

P, BAD = 4096, 1


def tables(**k):
    a = dict(new=P, ctx=P, s=2, pages=P, listed=9, window=0, sinks=0, pad=0, bt=P, width=4, qsl=P, seq=P, pos=P, slots=P, t=5,
             bs=16, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_build_step_tables(*{**a, **k}.values())


def test_step_tables_refuses_on_the_host():
    bad = [dict(s=-1), dict(t=-1), dict(listed=-1), dict(window=-1), dict(sinks=-1), dict(bs=32), dict(width=0),
           dict(width=(1 << 28) + 1), dict(s=(1 << 20) + 1), dict(new=None), dict(ctx=None), dict(pages=None), dict(bt=None), dict(qsl=None),
           dict(seq=None), dict(pos=None), dict(slots=None)]
    assert [k for k in bad if tables(**k) != BAD] == []


def norm_rope(**k):
    a = dict(q=P, q_st=1792, q_sh=128, k=P, k_st=256, k_sh=128, v=P, v_st=256, v_sh=128, qw=P, kw=P, w32=0, eps=1e-6, cos=P,
             cs=128, sin=P, sn=128, r32=0, out=P, o_st=1792, o_sh=128, kc=P, vc=P, c_slot=256, c_head=128, slots=64, map=P, t=5,
             h=14, hkv=2, d=128, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_qk_norm_rope_append(*{**a, **k}.values())


def test_norm_rope_refuses_on_the_host():
    assert norm_rope(t=0) == 0
    bad = [dict(t=-1), dict(h=15), dict(hkv=0), dict(d=96), dict(slots=0), *({n: None} for n in (
        "q", "k", "v", "qw", "kw", "cos", "sin", "out", "kc", "vc", "map"))]
    assert [k for k in bad if norm_rope(**k) != BAD] == []


def window(**k):
    a = dict(q=P, q_st=1792, q_sh=128, k=P, v=P, sb=8192, st=512, sh=128, nb=10, bt=P, bts=8, mb=8, qsl=P, seq=P, ctx=P,
             window=64, sinks=4, scale=0.1, out=P, o_st=1792, o_sh=128, s=2, t=0, mq=8, single=-1, h=14, hkv=2, d=128, bs=16,
             ws=P, columns=64, split=0, ranges=0, runs=1, stream=None)
    assert set(k) <= set(a)
    return _lib.lib().bvllm_paged_window_attention(*{**a, **k}.values())


def test_window_attention_refuses_on_the_host():
    assert window() == 0 and window(t=5, s=0) == 0 and window(t=5, mq=0) == 0  # nothing to do
    bad = [dict(h=15), dict(d=96), dict(bs=32), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
           dict(scale=float("inf")), dict(t=-1), dict(s=-1), dict(hkv=0), dict(window=0), dict(window=-5), dict(sinks=-1),
           dict(mq=-1), dict(single=-2)]
    assert [k for k in bad if window(**k) != BAD] == []
    bad = [dict(q=None), dict(out=None), dict(k=None), dict(qsl=None), dict(seq=None), dict(ctx=None), dict(bt=None),
           dict(q=P + 2), dict(out=P + 8), dict(q_st=1790), dict(o_sh=4), dict(sb=0), dict(sb=8190), dict(sb=1 << 31), dict(nb=0),
           dict(mb=0), dict(bts=7), dict(t=1 << 28), dict(st=1 << 28), dict(columns=16),
           dict(columns=256), dict(split=-1), dict(split=1 << 21, ranges=1), dict(split=1), dict(split=1, ranges=3), dict(ranges=1),
           dict(split=2, ranges=1, ws=None), dict(split=2, ranges=1, ws=P + 4), dict(runs=0), dict(runs=9), dict(runs=2, ws=None),
           dict(runs=2, ws=P + 8), dict(single=3), dict(s=40, single=17)]
    assert [k for k in bad if window(**{"t": 16, **k}) != BAD] == []


def plan(seqs, tokens, longest, single, heads, hkv, d, width, window, sinks):
    """(columns, split_tiles, num_ranges, row_runs, bytes of scratch)."""
    out = (ctypes.c_int32 * 4)(7, 7, 7, 7)
    rc = _lib.lib().bvllm_window_plan(seqs, tokens, longest, single, heads, hkv, d, width, window, sinks, out)
    if rc:
        assert rc == BAD and list(out) == [7] * 4
        return None
    return (*out, _lib.lib().bvllm_window_workspace_bytes(seqs, tokens, heads, d, out[2], out[3]))


def test_plans_fit_what_the_call_takes_and_their_scratch_is_bounded():
    scratch = lambda *a: plan(*a)[4]  # noqa: E731
    # A full decode batch and a full prompt are not cut; one row or a short turn behind a long window is.
    assert scratch(64, 64, 1, -1, 28, 4, 128, 1024, 4096, 4) == 0
    assert scratch(1, 8192, 8192, 0, 28, 4, 128, 512, 1024, 4) == 0
    assert scratch(1, 1, 1, -1, 28, 4, 128, 2048, 4096, 4) > 0 and scratch(1, 77, 77, 0, 28, 4, 128, 2048, 4096, 4) > 0
    assert scratch(1, 1, 1, -1, 28, 4, 128, 4, 2**31 - 1, 2**31 - 1) == 0  # a table of 4 pages
    # Nothing to do, or nothing that the call would take.
    for none in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        assert plan(*none, -1, 28, 4, 128, 64, 64, 4) == (128, 0, 0, 1, 0)
    for bad in ((-1, 1, 1, -1, 28, 4, 128, 64, 64, 4), (1, 1, 1, -1, 27, 4, 128, 64, 64, 4), (1, 1, 1, -1, 28, 4, 96, 64, 64, 4),
                (1, 1, 1, -1, 28, 4, 128, 0, 64, 4), (1, 1, 1, -1, 28, 4, 128, 64, 0, 4), (1, 1, 1, -1, 28, 4, 128, 64, 64, -1),
                (1, 1, -1, -1, 28, 4, 128, 64, 64, 4), (2, 9, 8, 3, 28, 4, 128, 64, 64, 4), (20, 9, 8, 10, 28, 4, 128, 64, 64, 4), (1, 1 << 28, 1, -1, 28, 4, 128, 64, 64, 4)):
        assert plan(*bad) is None
    rng = random.Random(0)
    taken = set()
    for _ in range(4000):
        seqs, longest = rng.randint(1, rng.choice([1, 8, 300])), rng.choice([1, 1, rng.randint(2, 100), rng.randint(2, 9000)])
        tokens = rng.randint(longest, longest * seqs)
        heads, hkv, d = rng.choice([(28, 4, 128), (14, 2, 64), (8, 8, 64), (40, 1, 128), (64, 64, 128)])
        width = rng.choice([1, 7, rng.randint(17, 700), 2049, 1 << 27])
        columns, split, ranges, runs, nbytes = plan(
            seqs, tokens, longest, rng.choice([-1, 0, rng.randint(0, min(seqs, tokens))]), heads, hkv, d, width,
            rng.choice([1, 40, 1024, 8192, 2**31 - 1]), rng.choice([0, 4, 300, 2**31 - 1]))
        assert 0 <= nbytes <= 129 << 20 and (nbytes > 0) == (split > 0 or runs > 1)
        assert 1 <= runs <= min(width, 4096) and columns in (128, 64, 32)
        assert ranges == 0 if split == 0 else 2 <= ranges <= -(-(-(-width // 4)) // split)
        taken.add((columns if longest > 1 else 0, split > 0, runs > 1))
    assert len(taken) >= 9, taken


def test_the_wrappers_refuse_tensors_of_the_cpu():
    from babyvllm.kernels.step_tables import build_step_tables

    v = torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm"):
        build_step_tables(v, v, v, 2, 2)
    from babyvllm.kernels.qk_norm_rope import fused_qk_norm_rope_and_cache
    from babyvllm.kernels.window_attn import paged_window_attention
    from babyvllm.worker.context import AttentionMetadata

    q, cache = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 16, 1, 64, dtype=torch.bfloat16)
    w = torch.ones(64)
    with pytest.raises(RuntimeError, match="ROCm"):
        fused_qk_norm_rope_and_cache(q, q[:, :1], q[:, :1], w, w, 1e-6, q[:, 0], q[:, 0], cache, torch.zeros(2).long())
    md = AttentionMetadata(None, v[:, None], torch.zeros(3, dtype=torch.int32), v, v, [0, 1, 2], [1, 1], [0, 0], 1, 1)
    with pytest.raises(RuntimeError, match="ROCm"):
        paged_window_attention(q, cache, md, 0.1, 4)


def test_no_access_to_registers_of_loads_in_flight(tmp_path):
    """As ``test_asm_hazards``, for the rows' page loads here."""
    import subprocess

    import build_lib
    from tests import asm_hazards

    if not build_lib.Path(build_lib.HIPCC).exists():
        pytest.skip("hipcc not available")
    out = tmp_path / "window_attn.s"
    res = subprocess.run([build_lib.HIPCC, *build_lib.FLAGS, "--cuda-device-only", "-S", "-o", str(out),
                          str(build_lib.CSRC / "window_attn.hip")], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    asm = out.read_text()
    names = asm_hazards.kernel_names(asm)
    assert names and "global_load_dwordx" in asm and ";;#ASMSTART" in asm
    hits = {n: asm_hazards.check_kernel(asm, n) for n in names}
    assert not any(hits.values()), {n[:70]: h[:3] for n, h in hits.items() if h}


@pytest.mark.parametrize("bad", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1)])
def test_a_layer_refuses_windows_that_are_none(bad):
    from babyvllm.layers.attention import Attention

    with pytest.raises(ValueError, match="window"):
        Attention(2, 64, 1, **bad)


def test_configs_leave_windows_and_head_norms_off():
    from babyvllm.config import qwen2_5_0_5b, qwen2_5_7b

    for cfg in (qwen2_5_7b(), qwen2_5_0_5b()):
        assert cfg.sliding_window is None and cfg.attention_sinks == 0 and cfg.qk_norm is False
