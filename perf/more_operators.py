"""The operators of a windowed serving step over the paged KV cache, as they are measured.

"tables":    block tables and slot maps from request lengths (babyvllm.kernels.step_tables)
"norm_rope": RMS norm of each query and key head, rotation and append (babyvllm.kernels.qk_norm_rope)
"window":    attention of a sliding window and a few first tokens (babyvllm.kernels.window_attn)

Shapes are the two presets of babyvllm.config: "7b" (28 query / 4 KV heads of 128) and "0.5b"
(14 / 2 heads of 64). Ragged lengths are geometric quantiles between two bounds, so they follow
from the case alone; their order, the pages and all values follow from the seed.
"""

import math
import os
import random
import sys
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
PAGE = 16
EPS = 1e-6
HEADS = {"7b": (28, 4, 128), "0.5b": (14, 2, 64)}  # query heads, KV heads, head size


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # One chat's decode step: all launch and latency.
        {"name": "tables_1", "op": "tables", "seqs": 1, "ones": 1, "ctx_lo": 500, "ctx_hi": 500, "new_lo": 1, "new_hi": 1,
         "pad": 0, "width": 129, "window": 0, "sinks": 0},
        # A full decode batch whose windowed caches dropped their old pages, padded to a graph's rows.
        {"name": "tables_50_windowed", "op": "tables", "seqs": 50, "ones": 50, "ctx_lo": 100, "ctx_hi": 20000, "new_lo": 1,
         "new_hi": 1, "pad": 14, "width": 0, "window": 1024, "sinks": 4},
        # Prompts beside a large decode batch, tables over the whole position range.
        {"name": "tables_512_mixed", "op": "tables", "seqs": 512, "ones": 400, "ctx_lo": 50, "ctx_hi": 32000, "new_lo": 31,
         "new_hi": 700, "pad": 0, "width": 2048, "window": 0, "sinks": 0},
        # A decode step of a few chats with the small model.
        {"name": "norm_rope_5", "op": "norm_rope", "shape": "0.5b", "tokens": 5, "rows": "bf16", "weight": "bf16"},
        # A full decode batch.
        {"name": "norm_rope_64", "op": "norm_rope", "shape": "7b", "tokens": 64, "rows": "bf16", "weight": "bf16"},
        # A step of prompts, rotation rows and weights in fp32.
        {"name": "norm_rope_8192", "op": "norm_rope", "shape": "7b", "tokens": 8192, "rows": "fp32", "weight": "fp32"},
        # One chat with the small model: all launch and latency.
        {"name": "window_1", "op": "window", "shape": "0.5b", "seqs": 1, "ones": 1, "ctx_lo": 700, "ctx_hi": 700,
         "new_lo": 1, "new_hi": 1, "window": 256, "sinks": 4},
        # A full decode batch, some chats shorter than the window, most longer.
        {"name": "window_64_decode", "op": "window", "shape": "7b", "seqs": 64, "ones": 64, "ctx_lo": 300, "ctx_hi": 16000,
         "new_lo": 1, "new_hi": 1, "window": 1024, "sinks": 4},
        # Long documents, a wide window, few users.
        {"name": "window_6_wide", "op": "window", "shape": "7b", "seqs": 6, "ones": 6, "ctx_lo": 20000, "ctx_hi": 32000,
         "new_lo": 1, "new_hi": 1, "window": 8192, "sinks": 64},
        # A few new tokens of one long chat behind a wide window.
        {"name": "window_1_turn", "op": "window", "shape": "7b", "seqs": 1, "ones": 0, "ctx_lo": 16000, "ctx_hi": 16000,
         "new_lo": 77, "new_hi": 77, "window": 4096, "sinks": 4},
        # Prompts of odd lengths beside decode rows.
        {"name": "window_30_mixed", "op": "window", "shape": "7b", "seqs": 30, "ones": 24, "ctx_lo": 100, "ctx_hi": 9000,
         "new_lo": 65, "new_hi": 1001, "window": 512, "sinks": 16},
        # One long prompt: the largest contraction.
        {"name": "window_1_prompt", "op": "window", "shape": "7b", "seqs": 1, "ones": 0, "ctx_lo": 0, "ctx_hi": 0,
         "new_lo": 8192, "new_hi": 8192, "window": 1024, "sinks": 4},
    ]


# No drawn case costs more than the largest listed one of its kind.
MAX_TABLE_BYTES = 5.2e6
MAX_TOKENS = 8192
MAX_WINDOW_FLOPS = 1.13e11
MAX_WINDOW_BYTES = 5e8  # as long as those products take
MAX_WINDOW_SCORES = 8192 * 28 * 8192  # of the plain form, which pads every sequence to the longest


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_lengths(rng, most_seqs, most_new):
    seqs = _log_int(rng, 1, most_seqs)
    # Decode steps, prompts, and both.
    ones = rng.choice([seqs, seqs, 0, rng.randint(0, seqs)])
    ctx_hi = 0 if rng.random() < 0.08 else _log_int(rng, 8, 32000)
    new_hi = _log_int(rng, 2, most_new)
    return {"seqs": seqs, "ones": ones,
            "ctx_lo": ctx_hi if rng.random() < 0.3 else (0 if ctx_hi == 0 else _log_int(rng, max(1, ctx_hi // 50), ctx_hi)),
            "ctx_hi": ctx_hi, "new_lo": _log_int(rng, max(1, new_hi // 20), new_hi), "new_hi": new_hi,
            "window": _log_int(rng, 16, 8192), "sinks": rng.choice([0, 1, 4, 4, 16, _log_int(rng, 1, 128)])}


def draw(rng):
    while True:
        op = rng.choice(["tables", "norm_rope", "window", "window", "window"])
        if op == "norm_rope":
            return {"op": op, "shape": rng.choice(["7b", "0.5b"]), "tokens": _log_int(rng, 1, MAX_TOKENS),
                    "rows": rng.choice(["bf16", "bf16", "fp32"]), "weight": rng.choice(["bf16", "fp32"])}
        if op == "tables":
            case = {"op": op, **_draw_lengths(rng, 512, 4096)}
            case["pad"] = rng.choice([0, 0, _log_int(rng, 1, 64)])
            case["width"] = rng.choice([0, 0, 2560])  # the widest row, or that of the longest request there can be
            if rng.random() < 0.5:
                case["window"] = case["sinks"] = 0
            if sum(_lengths(case)[1]) <= 4 * MAX_TOKENS and work(case)["bytes"] <= MAX_TABLE_BYTES:
                return case
        else:
            case = {"op": op, "shape": rng.choice(["7b", "7b", "0.5b"]), **_draw_lengths(rng, 64, 8192)}
            ctx, new = _lengths(case)
            keys = max(new) + min(max(ctx), case["window"] - 1 + case["sinks"])
            cost = work(case)
            if cost["flops"] <= MAX_WINDOW_FLOPS and cost["bytes"] <= MAX_WINDOW_BYTES and sum(new) <= MAX_TOKENS and \
                    case["seqs"] * max(new) * HEADS[case["shape"]][0] * keys <= MAX_WINDOW_SCORES:
                return case


def _spread(n, lo, hi):
    """n lengths from lo to hi at geometric quantiles (all hi when lo == hi)."""
    if lo == 0:
        return [0] * (n - n // 2) + [hi] * (n // 2)
    return [max(1, round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]


def _lengths(case):
    """(context, new tokens) of each sequence, before their order is drawn."""
    n, ones = case["seqs"], case["ones"]
    return _spread(n, case["ctx_lo"], case["ctx_hi"]), [1] * ones + _spread(n - ones, case["new_lo"], case["new_hi"])


def _held(case, ctx, new):
    """Table entries that a sequence holds: all, or with a window those of its first tokens and from the
    first page on that its first new token sees."""
    pages = -(-(ctx + new) // PAGE)
    if not case["window"]:
        return list(range(pages))
    kept = -(-case["sinks"] // PAGE)
    first = max(0, ctx - case["window"] + 1) // PAGE
    return [i for i in range(pages) if i < kept or i >= first]


def _seen_pairs(c, n, window, sinks):
    """Visible (row, key) pairs of n rows at positions c .. c + n - 1."""
    def below(p, w):  # sum of min(x, w) over x = 1 .. p
        return p * (p + 1) // 2 if p <= w else w * (w + 1) // 2 + (p - w) * w
    # Keys in the window, and first tokens before it: min(sinks, positions before the window).
    def first(p):  # sum over x = 1 .. p of min(sinks, max(0, x - window))
        return below(max(0, p - window), sinks)
    return below(c + n, window) - below(c, window) + first(c + n) - first(c)


def work(case):
    if case["op"] == "tables":
        ctx, new = _lengths(case)
        rows = sum(new) + case["pad"]
        held = sum(len(_held(case, c, n)) for c, n in zip(ctx, new))
        width = case["width"] or max(-(-(c + n) // PAGE) for c, n in zip(ctx, new))
        s = case["seqs"]
        return {"bytes": 8 * s + 4 * held + 4 * s * width + 4 * (2 * s + 1) + 16 * rows, "flops": 0}
    h, hkv, d = HEADS[case["shape"]]
    if case["op"] == "norm_rope":
        t = case["tokens"]
        rows = 2 * t * d * (2 if case["rows"] == "bf16" else 4)
        weights = 2 * d * (2 if case["weight"] == "bf16" else 4)
        return {"bytes": 2 * t * (h + 2 * hkv) * d * 2 + rows + weights + 8 * t, "flops": t * (h + hkv) * d * 7}
    ctx, new = _lengths(case)
    w, sinks, t = case["window"], case["sinks"], sum(new)
    # Orders of the two lists are independent: the sums below are their averages over the orders.
    n_avg = [(n, new.count(n) / len(new)) for n in sorted(set(new))]
    pairs = sum(f * _seen_pairs(c, n, w, sinks) for c in ctx for n, f in n_avg)
    # Keys that some row of the sequence sees.
    keys = sum(min(c, w - 1) + min(sinks, max(0, c - (w - 1))) for c in ctx) + t
    return {"bytes": 2 * keys * hkv * d * 2 + 2 * t * h * d * 2, "flops": 4 * d * h * pairs}


# ----------------------------------------------------------------- the inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed % (1 << 60))


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, dtype=torch.bfloat16, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _drawn_lengths(case, rng):
    ctx, new = _lengths(case)
    rng.shuffle(ctx)
    rng.shuffle(new)
    return ctx, new


def _prepare_tables(case, seed):
    rng = random.Random(seed)
    ctx, new = _drawn_lengths(case, rng)
    held = [_held(case, c, n) for c, n in zip(ctx, new)]
    order = list(range(sum(len(h) for h in held)))
    rng.shuffle(order)
    width = case["width"] or max(-(-(c + n) // PAGE) for c, n in zip(ctx, new))
    return SimpleNamespace(op="tables", new=_i32(new), ctx=_i32(ctx), pages=_i32(order),
                           rows=sum(new) + case["pad"], width=width, window=case["window"] or None, sinks=case["sinks"])


def _prepare_norm_rope(case, seed):
    h, hkv, d = HEADS[case["shape"]]
    t = case["tokens"]
    g = _gen(seed)
    pages = -(-t // PAGE) + 4
    # q, k and v are views of the step's fused projection, as the model gives them.
    qkv = _randn(g, t, (h + 2 * hkv) * d)
    kind = torch.bfloat16 if case["rows"] == "bf16" else torch.float32
    inv = 1e6 ** (-torch.arange(0, d, 2, device=DEV).double() / d)
    # Prompts' tokens are neighbours; tokens of a decode batch are anywhere.
    at = torch.arange(t, device=DEV) if t > 256 else torch.randint(0, 32768, (t,), device=DEV, generator=g)
    angle = at.double()[:, None] * torch.cat((inv, inv))
    weight = lambda: (1 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(  # noqa: E731
        torch.bfloat16 if case["weight"] == "bf16" else torch.float32)
    slots = torch.randperm(pages * PAGE, device=DEV, generator=g)[:t] if t <= 256 else \
        (torch.randperm(pages, device=DEV, generator=g)[:, None] * PAGE + torch.arange(PAGE, device=DEV)).view(-1)[:t]
    q, k, v = qkv.split([h * d, hkv * d, hkv * d], dim=-1)
    return SimpleNamespace(op="norm_rope", q=q.view(t, h, d), k=k.view(t, hkv, d), v=v.view(t, hkv, d),
                           q_weight=weight(), k_weight=weight(), cos=angle.cos().to(kind), sin=angle.sin().to(kind),
                           cache=_randn(g, 2, pages, PAGE, hkv, d), slots=slots.contiguous())


def _prepare_window(case, seed):
    h, hkv, d = HEADS[case["shape"]]
    rng = random.Random(seed)
    ctx, new = _drawn_lengths(case, rng)
    held = [_held(case, c, n) for c, n in zip(ctx, new)]
    total = sum(len(x) for x in held)
    order = list(range(total))
    rng.shuffle(order)
    width = max(-(-(c + n) // PAGE) for c, n in zip(ctx, new))
    tables = []
    for x in held:  # entries of pages that the sequence gave back are 0
        row = [0] * width
        for i in x:
            row[i] = order.pop()
        tables.append(row)
    qsl = [0]
    for n in new:
        qsl.append(qsl[-1] + n)
    seq = [c + n for c, n in zip(ctx, new)]
    md = SimpleNamespace(
        slot_mapping=None, block_tables=_i32(tables), query_start_loc=_i32(qsl), seq_lens=_i32(seq), context_lens=_i32(ctx),
        query_start_loc_cpu=qsl, seq_lens_cpu=seq, context_lens_cpu=ctx, max_query_len=max(new), max_seq_len=max(seq))
    g = _gen(seed)
    qkv = _randn(g, sum(new), h + 2 * hkv, d)
    return SimpleNamespace(op="window", q=qkv[:, :h], cache=_randn(g, 2, total, PAGE, hkv, d), md=md, scale=d ** -0.5,
                           window=case["window"], sinks=case["sinks"])


def prepare(case, seed):
    return {"tables": _prepare_tables, "norm_rope": _prepare_norm_rope, "window": _prepare_window}[case["op"]](case, seed)


# ------------------------------------------------------ the framework's calls


def _run_own(s):
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "baby-vllm_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    if s.op == "tables":
        from babyvllm.kernels.step_tables import build_step_tables
        return tuple(build_step_tables(s.new, s.ctx, s.pages, s.rows, s.width, window=s.window, sinks=s.sinks))
    if s.op == "norm_rope":
        from babyvllm.kernels.qk_norm_rope import fused_qk_norm_rope_and_cache
        q = fused_qk_norm_rope_and_cache(s.q, s.k, s.v, s.q_weight, s.k_weight, EPS, s.cos, s.sin, s.cache, s.slots)
        return q, s.cache
    from babyvllm.kernels.window_attn import paged_window_attention
    return paged_window_attention(s.q, s.cache, s.md, s.scale, s.window, s.sinks)


# ------------------------------------------------------------ the plain forms


def _plain_tables(s):
    new, ctx = s.new.long(), s.ctx.long()
    length = ctx + new
    pages = (length + PAGE - 1) // PAGE
    kept = -(-s.sinks // PAGE)
    # Entries from `kept` up to `first` are not in the list.
    first = torch.zeros_like(ctx) if s.window is None else (ctx - (s.window - 1)).clamp(min=0) // PAGE
    gone = (first - kept).clamp(min=0)
    start = torch.cumsum(pages - gone, 0) - (pages - gone)
    col = torch.arange(s.width, device=DEV)[None]
    there = (col < pages[:, None]) & ((col < kept) | (col >= first[:, None]))
    at = start[:, None] + torch.where(col < kept, col, col - gone[:, None])
    tables = torch.where(there, s.pages[at.clamp(0, s.pages.shape[0] - 1)], torch.zeros_like(s.pages[:1]))
    qsl = torch.cat((torch.zeros_like(new[:1]), torch.cumsum(new, 0)))
    row = torch.arange(s.rows, device=DEV)
    seq = (torch.searchsorted(qsl, row, right=True) - 1).clamp(max=new.shape[0] - 1)
    live = row < qsl[-1]
    pos = ctx[seq] + row - qsl[seq]
    entry = tables[seq, (pos // PAGE).clamp(max=s.width - 1)].long()
    return (tables, qsl.int(), length.int(), torch.where(live, pos, 0), torch.where(live, entry * PAGE + pos % PAGE, -1))


def _plain_norm_rope(s):
    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        half = x.shape[-1] // 2
        other = torch.cat((-x[..., half:], x[..., :half]), -1)
        return (x * s.cos.float()[:, None] + other * s.sin.float()[:, None]).to(torch.bfloat16)
    rows = s.cache.view(2, -1, *s.cache.shape[3:])
    rows[0, s.slots] = turned(s.k, s.k_weight)
    rows[1, s.slots] = s.v
    return turned(s.q, s.q_weight), s.cache


def _plain_window(s):
    md, q = s.md, s.q
    t, h, d = q.shape
    hkv = s.cache.shape[3]
    n, seqs = md.max_query_len, md.seq_lens.shape[0]
    # Rows of each sequence, padded to the longest one.
    first_row, last_row = md.query_start_loc[:-1, None].long(), md.query_start_loc[1:, None].long()
    i = torch.arange(n, device=DEV)[None]
    rows = torch.where(first_row + i < last_row, first_row + i, first_row)
    # Keys that some row of the sequence can see: its first tokens, and from the window of its first row on.
    ctx, length = md.context_lens[:, None].long(), md.seq_lens[:, None].long()
    keys = max(m - c + min(c, s.window - 1 + s.sinks) for c, m in zip(md.context_lens_cpu, md.seq_lens_cpu))
    begin = (ctx - (s.window - 1)).clamp(min=0)
    kept = torch.minimum(begin, torch.full_like(begin, s.sinks))
    x = torch.arange(keys, device=DEV)[None]
    pos = torch.where(x < kept, x, x - kept + begin)
    there = pos < length
    page = md.block_tables.long().gather(1, (pos // PAGE).clamp(max=md.block_tables.shape[1] - 1))
    slots = page * PAGE + pos % PAGE
    k = s.cache[0].reshape(-1, hkv, d)[slots].float().permute(0, 2, 3, 1).reshape(seqs * hkv, d, keys)
    v = s.cache[1].reshape(-1, hkv, d)[slots].float().permute(0, 2, 1, 3).reshape(seqs * hkv, keys, d)
    qs = q[rows].float().view(seqs, n, hkv, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs * hkv, -1, d)
    at = (ctx + i)[:, :, None]
    seen = there[:, None] & (pos[:, None] <= at) & ((pos[:, None] > at - s.window) | (pos[:, None] < s.sinks))
    score = torch.bmm(qs, k.contiguous()).view(seqs, hkv, n, h // hkv, keys) * s.scale
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(seqs * hkv, -1, keys), v.contiguous()).view(seqs, hkv, n, h // hkv, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(seqs, n, h, d)
    token = torch.arange(t, device=DEV)
    seq = torch.searchsorted(md.query_start_loc.long(), token, right=True) - 1
    return o[seq, token - md.query_start_loc[seq].long()].to(q.dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"tables": _plain_tables, "norm_rope": _plain_norm_rope, "window": _plain_window}[state.op](state)


# ------------------------------------------------------------------ in 64 bits


def _exact_norm_rope(s):
    cos, sin = s.cos.double(), s.sin.double()
    half = s.q.shape[2] // 2

    def rotated(x, weight):
        out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        for i in range(x.shape[1]):
            y = x[:, i].double()
            y = y / ((y ** 2).sum(-1, keepdim=True) / (2 * half) + EPS).sqrt() * weight.double()
            a, b = y[:, :half], y[:, half:]
            out[:, i, :half] = a * cos[:, :half] - b * sin[:, :half]
            out[:, i, half:] = b * cos[:, half:] + a * sin[:, half:]
        return out
    cache = s.cache.double()
    page, offset = s.slots // PAGE, s.slots % PAGE
    cache[0, page, offset] = rotated(s.k, s.k_weight)
    cache[1, page, offset] = s.v.double()
    return rotated(s.q, s.q_weight), cache


def _exact_window(s):
    md = s.md
    hkv = s.cache.shape[3]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    group = s.q.shape[1] // hkv
    for i, (c, n) in enumerate(zip(md.context_lens_cpu, md.seq_lens_cpu)):
        a, b = md.query_start_loc_cpu[i:i + 2]
        low = max(0, c - s.window + 1)
        where = torch.cat((torch.arange(min(s.sinks, low), device=DEV), torch.arange(low, n, device=DEV)))
        page = md.block_tables[i].long()[where // PAGE]
        keys, vals = s.cache[0][page, where % PAGE].double(), s.cache[1][page, where % PAGE].double()
        for r in range(a, b, 2048):  # rows at a time
            at = torch.arange(c + r - a, c + min(b, r + 2048) - a, device=DEV)[:, None]
            hidden = ~((where <= at) & ((at - where < s.window) | (where < s.sinks)))
            for head in range(s.q.shape[1]):
                w = s.q[r:r + at.shape[0], head].double() @ keys[:, head // group].T.contiguous() * s.scale
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                out[r:r + at.shape[0], head] = w @ vals[:, head // group].contiguous()
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None
    return {"norm_rope": _exact_norm_rope, "window": _exact_window}[case["op"]](prepare(case, seed))
