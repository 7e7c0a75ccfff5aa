"""The calls of a windowed step without a GPU: what the C entries and the wrappers refuse (nothing is
launched: the pointers below are never read)."""

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
           dict(width=(1 << 28) + 1), dict(new=None), dict(ctx=None), dict(pages=None), dict(bt=None), dict(qsl=None),
           dict(seq=None), dict(pos=None), dict(slots=None)]
    assert [k for k in bad if tables(**k) != BAD] == []


def test_the_wrappers_refuse_tensors_of_the_cpu():
    from babyvllm.kernels.step_tables import build_step_tables

    v = torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm"):
        build_step_tables(v, v, v, 2, 2)
