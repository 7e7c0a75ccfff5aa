"""RMS norm of query and key heads, rotation and append on the GPU, against the formula in 64 bits.

Bound. With y1, y2 the normalised values of a pair, the output o = y1 c1 - y2 s1 (or y2 c2 + y1 s2) is off by its own
rounding, at most 2^-8 |o|, and by fp32 arithmetic relative to |y1 c| + |y2 s|: the mean of D <= 256 squares is summed in
16 fmas of a lane and 4 steps across lanes, 20 * 2^-24, and half of that reaches its root; the root, the quotient, two
products of the norm and two of the rotation and their sum are off by at most 2^-24 (the root's library form 2^-23) each:
under 20 * 2^-24 in all. Values of bf16's subnormals are off by at most 2^-134.
"""

import pytest
import torch

from babyvllm.kernels.qk_norm_rope import fused_qk_norm_rope_and_cache

pytestmark = pytest.mark.gpu
PAGE = 16
BF16, FP32 = torch.bfloat16, torch.float32
EPS = 1e-6


def build(t, heads, hkv, d, rows=BF16, weight=BF16, seed=0, pages=None, magnitude=1.0, pad=0):
    """The step's projection, cut into q, k and v; `pad` columns behind them (odd ones leave rows unaligned)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = t // PAGE + 3 if pages is None else pages
    qkv = (magnitude * torch.randn(t, (heads + 2 * hkv) * d + pad, device="cuda", generator=g)).to(BF16)
    q, k, v, _ = qkv.split([heads * d, hkv * d, hkv * d, pad], dim=-1)
    angle = torch.randn(t, d // 2, device="cuda", generator=g, dtype=torch.float64) * 100
    angle = torch.cat((angle, angle), -1)
    w = [(1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(weight) for _ in range(2)]
    cache = torch.randn(2, pages, PAGE, hkv, d, device="cuda", generator=g).to(BF16)
    slots = torch.randperm(pages * PAGE, device="cuda", generator=g)[:t]
    return [q.view(t, heads, d), k.view(t, hkv, d), v.view(t, hkv, d), *w, EPS, angle.cos().to(rows), angle.sin().to(rows),
            cache, slots]


def rotated(x, w, eps, cos, sin):
    """(outputs, bound)."""
    x, w, cos, sin = x.double(), w.double(), cos.double()[:x.shape[0], None], sin.double()[:x.shape[0], None]
    half = x.shape[-1] // 2
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    a, b = y[..., :half], y[..., half:]
    parts = [(a * cos[..., :half], -b * sin[..., :half]), (b * cos[..., half:], a * sin[..., half:])]
    out = torch.cat([p + m for p, m in parts], -1)
    reach = torch.cat([p.abs() + m.abs() for p, m in parts], -1)
    return out, 2 ** -8 * out.abs() + 20 * 2 ** -24 * (1 + 2 ** -8) * reach + 2 ** -134


def near(got, want, what):
    out, tol = want
    diff = (got.double() - out).abs()
    assert torch.equal(torch.isnan(got), torch.isnan(out)), what
    diff = torch.nan_to_num(diff, nan=0.0)
    assert (diff <= torch.nan_to_num(tol, nan=0.0)).all(), (what, (diff / tol).max().item())


def check(args, **k):
    q, kk, v, qw, kw, eps, cos, sin, cache, slots = args
    before, kept = cache.clone(), [x.clone() for x in (q, kk, v)]
    got = fused_qk_norm_rope_and_cache(*args, **k)
    near(got, rotated(kept[0], qw, eps, cos, sin), "q")
    if "out" not in k:
        assert got.is_contiguous() and all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip((q, kk, v), kept))
    t = q.shape[0]
    there = (slots[:t] >= 0) & (slots[:t] < cache.shape[1] * PAGE)
    flat, old = cache.view(2, -1, *cache.shape[3:]), before.view(2, -1, *cache.shape[3:])
    at = slots[:t][there]
    out, tol = rotated(kept[1], kw, eps, cos, sin)
    near(flat[0, at], (out[there], tol[there]), "k")
    assert torch.equal(flat[1, at], kept[2][there])
    rest = torch.ones(flat.shape[1], dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(flat[:, rest], old[:, rest])
    return got


@pytest.mark.parametrize("weight", [BF16, FP32], ids=str)
@pytest.mark.parametrize("rows", [BF16, FP32], ids=str)
@pytest.mark.parametrize("heads,hkv,d", [(28, 4, 128), (14, 2, 64), (1, 1, 128), (8, 8, 64), (5, 1, 256), (16, 2, 256), (33, 11, 64)])
def test_against_the_formula(heads, hkv, d, rows, weight):
    for t in (1, 2, 5, 64, 131):
        check(build(t, heads, hkv, d, rows, weight, seed=t))


@pytest.mark.parametrize("pad", [1, 3, 4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_any_alignment(d, pad):
    args = build(9, 6, 2, d, pad=pad)
    check(args)
    # Views that start inside a row of cos, of a weight, of the values.
    cos = torch.randn(10, d + 3, device="cuda").to(BF16)
    args[6], args[7] = cos[:9, 1:d + 1], torch.randn(9, d + 1, device="cuda").to(BF16)[:, :d]
    args[3] = torch.randn(d + 1, device="cuda").to(BF16)[1:]
    check(args)


def test_a_long_step():
    check(build(8192, 28, 4, 128, FP32, FP32))


@pytest.mark.parametrize("magnitude", [0.0, 1e-30, 1e-4, 1e4, 1e15])
def test_magnitudes(magnitude):
    check(build(20, 7, 1, 128, FP32, FP32, magnitude=magnitude))


def test_values_that_are_not_finite_stay_in_their_head():
    args = build(4, 7, 1, 64)
    args[0][1, 3, 5] = float("nan")
    args[1][2, 0, 40] = float("nan")
    got = check(args)
    assert torch.isnan(got).any(-1).sum() == 1


def test_slots_outside_the_cache_are_not_written():
    args = build(12, 7, 1, 64, pages=2)
    args[9] = torch.tensor([-1, 0, 31, 32, 2**40, -2**60, 5, 6, 7, 8, 9, -1], device="cuda")
    check(args)


def test_more_rows_and_slots_than_tokens():
    args = build(12, 7, 1, 64)
    wide = build(20, 7, 1, 64, seed=1)
    args[6], args[7] = wide[6], wide[7]
    args[9] = torch.cat((args[9], args[9].new_full((8,), 10**9)))
    check(args)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_in_place_and_given_outputs(d):
    args = build(30, 9, 3, d)
    want = check(args)
    out = torch.full((30, 9, d + 8), 7.0, device="cuda", dtype=BF16)
    assert check(args, out=out[..., :d]).data_ptr() == out.data_ptr()
    assert torch.equal(out[..., :d], want) and (out[..., d:] == 7).all()
    args = build(30, 9, 3, d)
    kept = [x.clone() for x in args[1:3]]
    q = args[0]
    assert check(args, out=q) is q and torch.equal(q, want)
    assert torch.equal(args[1], kept[0]) and torch.equal(args[2], kept[1])


def test_a_cache_past_2_31_elements():
    pages = 2**31 // (PAGE * 8 * 128) + 9
    args = build(5, 8, 8, 128, pages=1)
    args[8] = torch.zeros(2, pages, PAGE, 8, 128, device="cuda", dtype=BF16)
    args[9] = torch.tensor([0, pages * PAGE - 1, pages * PAGE // 2, pages * PAGE - 17, 5], device="cuda")
    check(args)


def test_captured_and_on_another_stream():
    args = build(16, 14, 2, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = fused_qk_norm_rope_and_cache(*args)
    side.synchronize()
    near(first, rotated(args[0], args[3], EPS, args[6], args[7]), "q")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fused_qk_norm_rope_and_cache(*args)
    for i in range(3):
        args[0].copy_(torch.randn_like(args[0]))
        args[9].copy_(torch.randperm(args[8].shape[1] * PAGE, device="cuda")[:16])
        args[8].zero_()
        graph.replay()
        torch.cuda.synchronize()
        cache = args[8].clone()
        args[8].zero_()
        assert torch.equal(check(args), got) and torch.equal(args[8], cache)


def test_refusals():
    args = build(6, 8, 2, 64)

    def call(error, match=None, out=None, **k):
        names = ["q", "k", "v", "q_weight", "k_weight", "eps", "cos", "sin", "cache", "slots"]
        given = [k.pop(n, a) for n, a in zip(names, args)]
        assert not k
        with pytest.raises(error, match=match):
            fused_qk_norm_rope_and_cache(*given, out=out)

    q, k, v, qw, kw, _, cos, sin, cache, slots = args
    call(TypeError, q=q.float())
    call(ValueError, q=q[..., :48], k=k[..., :48], v=v[..., :48])
    call(ValueError, k=k[:5])
    call(ValueError, v=v[:, :1])
    call(ValueError, q=q.transpose(1, 2))
    call(TypeError, q_weight=qw.float())
    call(TypeError, q_weight=qw.half(), k_weight=kw.half())
    call(ValueError, q_weight=qw[:32], k_weight=kw[:32])
    call(TypeError, cos=cos.float())
    call(ValueError, cos=cos[:3], sin=sin[:3])
    call(ValueError, cache=cache[:, :, :, :1])
    call(ValueError, cache=cache.transpose(2, 3).contiguous().transpose(2, 3))
    call(TypeError, cache=cache.float())
    call(TypeError, slots=slots.int())
    call(TypeError, slots=slots[:5])
    call(RuntimeError, "ROCm", sin=sin.cpu())
    call(ValueError, "out", out=torch.empty(6, 8, 64, device="cuda"))
    call(ValueError, "out", out=torch.empty(6, 8, 32, device="cuda", dtype=BF16))
    call(ValueError, "memory", out=torch.empty(1, 8, 64, device="cuda", dtype=BF16).expand(6, 8, 64))
    room = torch.empty(7, 8, 64, device="cuda", dtype=BF16)
    call(ValueError, "memory", q=room[:6], out=room[1:])
    assert fused_qk_norm_rope_and_cache(q[:0], k[:0], v[:0], *args[3:]).shape == (0, 8, 64)
