"""How many bits the softmax weights of window attention keep: 16 in single rows.

Bound. A weight P enters the second product as two bf16 operands: its upper 16 bits, which leave less than 2^-7 of it, and
what they leave, off by at most 2^-8 of that: 2^-15 of P. With the scores' own error (fp32 sums of D <= 128 products of q and
k, D * 2^-24 of their magnitudes, times the scale: under 2^-13 here, and the exponent's roundings, under 2^-20 at these sizes)
d = 2^-15 + 2^-13 + 2^-20, the output is off by at most d / (1 - d) * sum_j w_j |v_j| (sum_j w_j |v_j - o| where the
weights' sum has the same errors: the larger of both is taken), by fp32 sums, n * 2^-23 * sum_j w_j |v_j|, and by its own
rounding, 2^-8 |o|. With weights of one operand (d = 2^-8) outputs near zero leave this bound.
"""

import pytest
import torch

from babyvllm.kernels.window_attn import paged_window_attention
from tests._cases import python_path
from tests.test_window_attn_gpu import build, raw_call, run

pytestmark = pytest.mark.gpu
PAGE = 16
HEADS = [(2, 7, 128), (2, 7, 64), (1, 1, 128), (1, 20, 64)]


def bounded(q, cache, md, scale, window, sinks):
    """(outputs, bound) in 64 bits."""
    group = q.shape[1] // cache.shape[3]
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    tables, qsl = md.block_tables.tolist(), md.query_start_loc.tolist()
    d = 2 ** -15 + 2 ** -13 + 2 ** -20
    for s, ctx in enumerate(md.context_lens.tolist()):
        for r in range(qsl[s], qsl[s + 1]):
            p = ctx + r - qsl[s]
            sees = torch.tensor([j for j in range(p + 1) if j > p - window or j < sinks], device=q.device)
            page = torch.tensor(tables[s], device=q.device)[sees // PAGE]
            k, v = (c[page, sees % PAGE].double().repeat_interleave(group, 1) for c in (cache[0], cache[1]))  # [n, H, D]
            x = q[r].double()
            assert q.shape[2] * 2 ** -24 * scale * (k * x).abs().sum(-1).max().item() < 2 ** -13
            w = torch.softmax((k * x).sum(-1) * scale, 0)[..., None]
            o = (w * v).sum(0)
            reach = (w * v.abs()).sum(0)
            out[r] = o
            tol[r] = d / (1 - d) * torch.maximum((w * (v - o).abs()).sum(0), reach) + len(sees) * 2 ** -23 * reach + 2 ** -8 * o.abs()
    return out, tol


def check(got, want, rows=slice(None)):
    out, tol = want[0][rows], want[1][rows]
    diff = (got[rows].double() - out).abs()
    assert (diff <= tol).all(), f"off by up to {(diff / tol).max().item():.3g} times the bound"


ROWS = [(c, 1) for c in (0, 3, 16, 40, 100, 150, 300, 700, 1500)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_single_rows(heads):
    for window, sinks in ((40, 4), (256, 0), (1000, 20)):
        q, cache, md = build(ROWS, *heads, window, sinks)
        want = bounded(q, cache, md, 0.1, window, sinks)
        for runs in (1, 2, 5):
            check(raw_call(q, cache, md, 0.1, window, sinks, 128, 0, runs), want)
        check(paged_window_attention(q, cache, md, 0.1, window, sinks), want)


@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_few_rows_of_wide_windows(heads, monkeypatch):
    q, cache, md = build([(5000, 1), (900, 1)], *heads, 4096, 4)
    want = bounded(q, cache, md, 0.1, 4096, 4)
    check(paged_window_attention(q, cache, md, 0.1, 4096, 4), want)
    python_path(monkeypatch)
    check(paged_window_attention(q, cache, md, 0.1, 4096, 4), want)


@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_single_rows_beside_prompts(heads):
    q, cache, md = build([(300, 1), (64, 9), (90, 1), (1000, 1), (0, 40)], *heads, 128, 4)
    want = bounded(q, cache, md, 0.1, 128, 4)
    for columns, split, runs in ((128, 0, 1), (64, 0, 3), (32, 1, 1)):
        check(raw_call(q, cache, md, 0.1, 128, 4, columns, split, runs), want, [0, 10, 11])


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("heads", [(2, 7, 128), (2, 7, 64)], ids=str)
def test_a_weight_of_one_meets_values_that_are_not_finite(heads, value):
    # Every row sees its own key alone: its weight is 1, of which the upper half leaves nothing.
    q, cache, md = build([(300, 1), (20, 1), (0, 1), (15, 70), (64, 3)], *heads, 1, 0)
    for s, (c, n) in enumerate(zip(md.context_lens_cpu, md.seq_lens_cpu)):
        for p in {c, n - 1}:
            cache[1, int(md.block_tables[s, p // PAGE]), p % PAGE, :, (5 * s + p) % heads[2]] = value
    run(q, cache, md, 1, 0, forms=[(128, 0, 1), (64, 0, 1), (32, 0, 2), (32, 1, 1)])
