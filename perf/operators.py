"""The operators that decode several candidates of a request over the paged KV cache, as they are measured.

"tree":    attention of a tree of drafted tokens over the cache (babyvllm.kernels.tree_attn)
"commit":  the tree's verified path, its K/V moved behind the context (babyvllm.kernels.tree_commit)
"select":  beam search's selection over beams and vocabulary (babyvllm.kernels.beam)
"reorder": the beams' block tables and cache pages after it (babyvllm.kernels.beam)

Shapes are the two presets of babyvllm.config: "7b" (28 query / 4 KV heads of 128, 28 layers,
152,064 tokens) and "0.5b" (14 / 2 heads of 64, 24 layers, 151,936 tokens). Ragged lengths are
geometric quantiles between two bounds, so they follow from the case alone; their order, the
pages, the trees and all values follow from the seed.
"""

import math
import os
import random
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 16
WORD = 64
HEADS = {"7b": (28, 4, 128, 28), "0.5b": (14, 2, 64, 24)}  # query heads, KV heads, head size, layers


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # One chat with a small model and a small draft: all launch and latency.
        {"name": "tree_1_small", "op": "tree", "shape": "0.5b", "seqs": 1, "ctx_lo": 300, "ctx_hi": 300,
         "new_lo": 8, "new_hi": 8, "branch": 3},
        # A serving batch with short chains (each draft token follows the one before it).
        {"name": "tree_48_chains", "op": "tree", "shape": "7b", "seqs": 48, "ctx_lo": 200, "ctx_hi": 4000,
         "new_lo": 2, "new_hi": 7, "branch": 1},
        # A few chats with mid-sized trees of different sizes.
        {"name": "tree_8_chats", "op": "tree", "shape": "7b", "seqs": 8, "ctx_lo": 500, "ctx_hi": 3000,
         "new_lo": 11, "new_hi": 45, "branch": 6},
        # One long document, one user, one tree.
        {"name": "tree_1_long", "op": "tree", "shape": "7b", "seqs": 1, "ctx_lo": 32000, "ctx_hi": 32000,
         "new_lo": 25, "new_hi": 25, "branch": 5},
        # Wide trees over long chats: the largest contraction.
        {"name": "tree_16_wide", "op": "tree", "shape": "7b", "seqs": 16, "ctx_lo": 1000, "ctx_hi": 8000,
         "new_lo": 64, "new_hi": 64, "branch": 12},
        # The smallest commit: one sequence, a few rows of every layer.
        {"name": "commit_1", "op": "commit", "shape": "0.5b", "seqs": 1, "ctx_lo": 300, "ctx_hi": 300,
         "new_lo": 8, "new_hi": 8, "branch": 3, "accept": 0.75},
        # A serving batch's commit, every layer of the larger model.
        {"name": "commit_48", "op": "commit", "shape": "7b", "seqs": 48, "ctx_lo": 200, "ctx_hi": 4000,
         "new_lo": 20, "new_hi": 64, "branch": 8, "accept": 0.8},
        # One request of four beams.
        {"name": "select_1x4", "op": "select", "groups": 1, "beams": 4, "candidates": 8, "vocab": 151936,
         "dtype": "bf16"},
        # An odd vocabulary in fp32 (rows that are not 16-byte aligned), odd beams.
        {"name": "select_6x5_odd", "op": "select", "groups": 6, "beams": 5, "candidates": 10, "vocab": 50257,
         "dtype": "fp32"},
        # A full batch of beams over the larger vocabulary.
        {"name": "select_16x8", "op": "select", "groups": 16, "beams": 8, "candidates": 16, "vocab": 152064,
         "dtype": "bf16"},
        # One request of four beams in the larger model: its partial pages, every layer.
        {"name": "reorder_1x4", "op": "reorder", "shape": "7b", "groups": 1, "beams": 4, "len_lo": 1003,
         "len_hi": 1003},
        # A full batch of beams.
        {"name": "reorder_16x8", "op": "reorder", "shape": "7b", "groups": 16, "beams": 8, "len_lo": 200,
         "len_hi": 2000},
    ]


# No drawn case costs more than the largest listed one of its kind: flops and padded scores of a
# tree, moved bytes of a commit or reorder, logits of a selection.
MAX_TREE_FLOPS = 5e10
MAX_TREE_SCORES = 16 * 64 * 28 * 8064
MAX_SEQS = 48
MAX_COMMIT_BYTES = 2.1e7
MAX_LOGIT_BYTES = 16 * 8 * 152064 * 2
MAX_BEAM_ROWS = 16 * 8


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_tree(rng, op):
    ctx_hi = 0 if rng.random() < 0.05 else _log_int(rng, 32, 32768)
    new_hi = _log_int(rng, 1, 160)
    case = {"op": op, "shape": rng.choice(["7b", "7b", "0.5b"]), "seqs": _log_int(rng, 1, MAX_SEQS),
            "ctx_lo": ctx_hi if rng.random() < 0.3 else (0 if ctx_hi == 0 else _log_int(rng, max(1, ctx_hi // 50), ctx_hi)),
            "ctx_hi": ctx_hi, "new_lo": _log_int(rng, 1, new_hi), "new_hi": new_hi, "branch": rng.choice([1, 2, 4, 8, 16])}
    if op == "commit":
        case["new_hi"] = min(64, case["new_hi"])
        case["new_lo"] = min(case["new_lo"], case["new_hi"])
        case["accept"] = rng.choice([0.3, 0.6, 0.8, 0.95])
    return case


def draw(rng):
    while True:
        op = rng.choice(["tree", "tree", "tree", "commit", "select", "select", "reorder"])
        if op == "tree":
            case = _draw_tree(rng, op)
            h = HEADS[case["shape"]][0]
            if work(case)["flops"] <= MAX_TREE_FLOPS and \
                    case["seqs"] * case["new_hi"] * h * (case["ctx_hi"] + case["new_hi"]) <= MAX_TREE_SCORES:
                return case
        elif op == "commit":
            case = _draw_tree(rng, op)
            if work(case)["bytes"] <= MAX_COMMIT_BYTES:
                return case
        elif op == "select":
            beams = _log_int(rng, 1, 32)
            dtype = rng.choice(["bf16", "bf16", "fp32"])
            vocab = rng.choice([151936, 152064, 32000, 50257, _log_int(rng, 100, 160000)])
            groups = _log_int(rng, 1, 16)
            case = {"op": op, "groups": groups, "beams": beams, "candidates": rng.choice([beams, 2 * beams]),
                    "vocab": vocab, "dtype": dtype}
            if groups * beams * vocab * (2 if dtype == "bf16" else 4) <= MAX_LOGIT_BYTES:
                return case
        else:
            hi = _log_int(rng, 1, 4000)
            case = {"op": op, "shape": rng.choice(["7b", "0.5b"]), "groups": _log_int(rng, 1, 16),
                    "beams": _log_int(rng, 2, 32), "len_lo": _log_int(rng, max(1, hi // 10), hi), "len_hi": hi}
            if case["groups"] * case["beams"] <= MAX_BEAM_ROWS:
                return case


def _spread(n, lo, hi):
    """n lengths from lo to hi at geometric quantiles (all hi when lo == hi)."""
    if lo == 0:
        return [0] * (n - n // 2) + [hi] * (n // 2)
    return [max(1, round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)]


def _lengths(case):
    """(context, new tokens) of each sequence, before their order is drawn."""
    n = case["seqs"]
    return _spread(n, case["ctx_lo"], case["ctx_hi"]), _spread(n, case["new_lo"], case["new_hi"])


def work(case):
    if case["op"] == "select":
        rows = case["groups"] * case["beams"]
        n = rows * case["vocab"]
        out = case["groups"] * case["candidates"] * 20
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + rows * 4 + out, "flops": 4 * n}
    h, hkv, d, layers = HEADS[case["shape"]]
    row = 2 * hkv * d * 2 * layers  # K and V of one token, every layer
    if case["op"] == "reorder":
        lens = _spread(case["groups"], case["len_lo"], case["len_hi"])
        k = case["beams"]
        # Half of the beams come from another one (see _parents), whose partial page is read and written.
        moved = sum(n % PAGE for n in lens) * k / 2
        tables = sum(n // PAGE for n in lens) * k * 4
        return {"bytes": 2 * (moved * row + tables), "flops": 0}
    ctx, new = _lengths(case)
    if case["op"] == "commit":
        a = case["accept"]
        rows = sum(sum(a ** i for i in range(1, min(n, 8))) for n in new)  # accepted behind the root
        return {"bytes": 2 * rows * row + sum(new) * 20, "flops": 0}
    t, w = sum(new), -(-case["new_hi"] // WORD)
    # Orders of the two lists are independent: the sums below are their averages over the orders.
    keys = sum(ctx) + t
    pairs = sum(ctx) * t / case["seqs"] + sum(n * (n + 1) / 2 for n in new)
    return {"bytes": 2 * keys * hkv * d * 2 + 2 * t * h * d * 2 + t * w * 8, "flops": 4 * d * h * pairs}


# ----------------------------------------------------------------- the inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed % (1 << 60))


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, dtype=torch.bfloat16, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tree(rng, n, branch):
    """Parents of n drafted tokens, root first; `branch` 1 is a chain."""
    return [-1] + [rng.randrange(max(0, i - branch), i) for i in range(1, n)]


def _ancestor_words(parents, words):
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    signed = lambda v: v - (1 << WORD) if v >> (WORD - 1) else v  # noqa: E731
    return [[signed(r >> (WORD * w) & ((1 << WORD) - 1)) for w in range(words)] for r in rows]


def _draft(case, seed):
    """The step's sequences: order of the lengths, trees, and what the runner knows on the host."""
    rng = random.Random(seed)
    ctx, new = _lengths(case)
    rng.shuffle(ctx)
    rng.shuffle(new)
    parents = [_tree(rng, n, case["branch"]) for n in new]
    qsl = [0]
    for n in new:
        qsl.append(qsl[-1] + n)
    seq = [c + n for c, n in zip(ctx, new)]
    words = -(-max(new) // WORD)
    mask = [w for p in parents for w in _ancestor_words(p, words)]
    md = SimpleNamespace(
        query_start_loc=_i32(qsl), seq_lens=_i32(seq), context_lens=_i32(ctx), query_start_loc_cpu=qsl,
        seq_lens_cpu=seq, context_lens_cpu=ctx, max_query_len=max(new), max_seq_len=max(seq),
        tree_mask=torch.tensor(mask, dtype=torch.int64, device=DEV))
    return rng, ctx, new, parents, md


def _prepare_tree(case, seed):
    h, hkv, d, _ = HEADS[case["shape"]]
    rng, ctx, new, parents, md = _draft(case, seed)
    pages = [-(-n // PAGE) for n in md.seq_lens_cpu]
    order = list(range(sum(pages) + 8))
    rng.shuffle(order)
    tables = []
    for n in pages:
        tables.append([order.pop() for _ in range(n)] + [0] * (max(pages) - n))
    md.block_tables = _i32(tables)
    g = _gen(seed)
    # q is a view of the step's fused projection, as the model gives it.
    qkv = _randn(g, sum(new), h + 2 * hkv, d)
    return SimpleNamespace(op="tree", q=qkv[:, :h], cache=_randn(g, 2, sum(pages) + 8, PAGE, hkv, d), md=md,
                           scale=d ** -0.5)


def _prepare_commit(case, seed):
    _, hkv, d, layers = HEADS[case["shape"]]
    rng, ctx, new, parents, md = _draft(case, seed)
    # Pages of the drafted tokens are the sequence's own; those of the context before them,
    # which a commit does not touch, come from a pool of 64.
    owned = [(c + n - 1) // PAGE - c // PAGE + 1 for c, n in zip(ctx, new)]
    pool = 64 + sum(n // PAGE + 2 for n in new)  # the most they can own
    order = list(range(64, pool))
    rng.shuffle(order)
    width = max(-(-n // PAGE) for n in md.seq_lens_cpu)
    tables = []
    for c, k in zip(ctx, owned):
        t = [rng.randrange(64) for _ in range(c // PAGE)] + [order.pop() for _ in range(k)]
        tables.append(t + [0] * (width - len(t)))
    md.block_tables = _i32(tables)
    # The model answers with the drafted child (one of them) with probability `accept`.
    draft, target = [], []
    for par in parents:
        tokens = [rng.randrange(150000) for _ in par]
        answer = [150000 + rng.randrange(1000) for _ in par]
        children = [[c for c, p in enumerate(par) if p == i] for i in range(len(par))]
        cur, depth = 0, 1
        while children[cur] and depth < 8 and rng.random() < case["accept"]:
            nxt = rng.choice(children[cur])
            answer[cur] = tokens[nxt]
            cur, depth = nxt, depth + 1
        draft += tokens
        target += answer
    caches = _randn(_gen(seed), layers, 2, pool, PAGE, hkv, d)
    return SimpleNamespace(op="commit", stack=caches, caches=list(caches.unbind(0)), md=md,
                           draft=torch.tensor(draft, device=DEV), target=torch.tensor(target, device=DEV),
                           parents=_i32([p for t in parents for p in t]))


def _prepare_select(case, seed):
    g = _gen(seed)
    rows = case["groups"] * case["beams"]
    # A language model's logits: a few tokens stand out of a broad rest, more so in some rows.
    x = torch.randn(rows, case["vocab"], device=DEV, generator=g)
    x = x * (1.5 + 2 * torch.rand(rows, 1, device=DEV, generator=g))
    x = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    scores = -torch.rand(rows, device=DEV, generator=g) * 3 - 20
    return SimpleNamespace(op="select", logits=x, scores=scores, beams=case["beams"], n=case["candidates"])


def _parents(rng, groups, k):
    """Parents of the surviving beams: half of them stay, the others continue a better one."""
    out = []
    for _ in range(groups):
        p = list(range(k))
        for b in rng.sample(range(k), k // 2):
            p[b] = rng.choice([q for q in range(k) if q != b])
        out.append(p)
    return out


def _prepare_reorder(case, seed):
    _, hkv, d, layers = HEADS[case["shape"]]
    rng = random.Random(seed)
    groups, k = case["groups"], case["beams"]
    lens = _spread(groups, case["len_lo"], case["len_hi"])
    rng.shuffle(lens)
    # The page being filled is a beam's own; full pages, which are shared, come from a pool of 64.
    order = list(range(64, 64 + groups * k))
    rng.shuffle(order)
    width = max(lens) // PAGE + 1
    tables = []
    for n in lens:
        for _ in range(k):
            t = [rng.randrange(64) for _ in range(n // PAGE)] + [order.pop()]
            tables.append(t + [0] * (width - len(t)))
    caches = _randn(_gen(seed), layers, 2, 64 + groups * k, PAGE, hkv, d)
    return SimpleNamespace(op="reorder", stack=caches, caches=list(caches.unbind(0)), tables=_i32(tables),
                           lens=_i32([n for n in lens for _ in range(k)]),
                           beams=torch.tensor(_parents(rng, groups, k), device=DEV))


def prepare(case, seed):
    return {"tree": _prepare_tree, "commit": _prepare_commit, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["op"]](case, seed)


# ------------------------------------------------------ the framework's calls


def _run_own(s):
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "baby-vllm_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    if s.op == "tree":
        from babyvllm.kernels.tree_attn import paged_tree_attention
        return paged_tree_attention(s.q, s.cache, s.md, s.scale)
    if s.op == "commit":
        from babyvllm.kernels.tree_commit import commit_draft_tree
        path, accepted, following = commit_draft_tree(s.caches, s.md, s.draft, s.target, s.parents)
        return path, accepted, following, s.stack
    from babyvllm.kernels.beam import beam_select, reorder_beams
    if s.op == "select":
        return beam_select(s.logits, s.scores, s.beams, s.n)
    reorder_beams(s.caches, s.tables, s.lens, s.beams)
    return s.tables, s.stack


# ------------------------------------------------------------ the plain forms


def _rows_of(md):
    """(row of the i-th token of each sequence [S, N], whether there is one)."""
    first, last = md.query_start_loc[:-1, None].long(), md.query_start_loc[1:, None].long()
    i = torch.arange(md.max_query_len, device=DEV)[None]
    valid = first + i < last
    return torch.where(valid, first + i, first.clamp(max=int(md.query_start_loc_cpu[-1]) - 1)), valid


def _plain_tree(s):
    md, q = s.md, s.q
    t, h, d = q.shape
    hkv = s.cache.shape[3]
    n, length, seqs = md.max_query_len, md.max_seq_len, md.seq_lens.shape[0]
    rows, _ = _rows_of(md)
    pos = torch.arange(length, device=DEV)
    slots = md.block_tables[:, pos // PAGE].long() * PAGE + pos % PAGE
    k = s.cache[0].reshape(-1, hkv, d)[slots].float().permute(0, 2, 3, 1).reshape(seqs * hkv, d, length)
    v = s.cache[1].reshape(-1, hkv, d)[slots].float().permute(0, 2, 1, 3).reshape(seqs * hkv, length, d)
    qs = q[rows].float().view(seqs, n, hkv, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs * hkv, -1, d)
    # Keys of the context are visible to all; a drafted one where its bit is set.
    j = pos[None] - md.context_lens[:, None].long()
    words = md.tree_mask[rows].gather(2, (j.clamp(min=0) // WORD).clamp(max=md.tree_mask.shape[1] - 1)[:, None].expand(-1, n, -1))
    seen = (j[:, None] < 0) | ((words >> (j[:, None].clamp(min=0) % WORD)) & 1 == 1)
    seen &= (pos[None] < md.seq_lens[:, None])[:, None]
    score = torch.bmm(qs, k.contiguous()).view(seqs, hkv, n, h // hkv, length) * s.scale
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(seqs * hkv, -1, length), v.contiguous()).view(seqs, hkv, n, h // hkv, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(seqs, n, h, d)
    token = torch.arange(t, device=DEV)
    seq = torch.searchsorted(md.query_start_loc.long(), token, right=True) - 1
    return o[seq, token - md.query_start_loc[seq].long()].to(q.dtype)


def _plain_commit(s):
    md = s.md
    n = md.max_query_len
    rows, valid = _rows_of(md)
    par = s.parents[rows].long()
    node = torch.arange(n, device=DEV)
    # A node is right where its token is its parent's answer and no sibling before it is.
    answer = s.target[rows].gather(1, par.clamp(min=0))
    right = valid & (par >= 0) & (s.draft[rows] == answer)
    before = (par[:, :, None] == par[:, None, :]) & (node[None, :] < node[:, None]) & right[:, None, :]
    right &= ~before.any(-1)
    # It is accepted where it and all its ancestors behind the root are right.
    bits = (md.tree_mask[rows][:, :, node // WORD] >> (node % WORD)) & 1 == 1
    ok = valid & (~(bits & (node > 0)) | right[:, None, :]).all(-1)
    accepted = ok.sum(-1)
    path = torch.where(ok, node, n).sort(-1).values
    last = path.gather(1, accepted[:, None] - 1)
    following = s.target[rows].gather(1, last)[:, 0]
    path = torch.where(path < n, path, -1)
    # Places behind the path stand for the root, which stays where it is.
    ctx = md.context_lens[:, None].long()
    source, dest = ctx + path.clamp(min=0), ctx + node
    width = md.block_tables.shape[1]
    slot = lambda p: md.block_tables.long().gather(1, (p // PAGE).clamp(max=width - 1)) * PAGE + p % PAGE  # noqa: E731
    live = node < accepted[:, None]
    moved_from, moved_to = slot(torch.where(live, source, ctx)), slot(torch.where(live, dest, ctx))
    flat = s.stack.view(*s.stack.shape[:2], -1, *s.stack.shape[4:])
    flat[:, :, moved_to.reshape(-1)] = flat[:, :, moved_from.reshape(-1)]
    return path.int(), accepted.int(), following, s.stack


def _plain_select(s):
    k, n = s.beams, s.n
    rows, vocab = s.logits.shape
    x = s.logits.float() + 0.0
    wide = s.logits.double()
    base = s.scores.double() - torch.logsumexp(wide, -1)
    # The n best of a row, equal ones by their index: the value's order and the index in one key.
    bits = x.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff))
    best = (order * (1 << 31) + ((1 << 31) - 1 - torch.arange(vocab, device=DEV))).topk(min(n, vocab), -1).values
    token = (1 << 31) - 1 - (best & ((1 << 31) - 1))
    total = (wide.gather(1, token) + base[:, None]).view(rows // k, -1)
    beam = torch.arange(k, device=DEV).repeat_interleave(token.shape[1])
    total, at = total.sort(dim=-1, descending=True, stable=True)
    return (total[:, :n].float().contiguous(), beam[at[:, :n]],
            token.view(rows // k, -1).gather(1, at[:, :n]))


def _plain_reorder(s):
    groups, k = s.beams.shape
    width = s.tables.shape[1]
    source = (torch.arange(groups, device=DEV)[:, None] * k + s.beams).view(-1)
    full = (s.lens // PAGE).long()
    col = torch.arange(width, device=DEV)
    # The page being filled is copied from the parent's, its first tokens.
    own_page = s.tables.gather(1, full.clamp(max=width - 1)[:, None])[:, 0].long()
    from_page = own_page[source]
    filled = torch.arange(PAGE, device=DEV) < (s.lens % PAGE)[:, None]
    s.stack[:, :, own_page] = torch.where(filled[None, None, :, :, None, None], s.stack[:, :, from_page],
                                          s.stack[:, :, own_page])
    s.tables.copy_(torch.where(col[None] < full[:, None], s.tables[source], s.tables))
    return s.tables, s.stack


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "commit": _plain_commit, "select": _plain_select,
            "reorder": _plain_reorder}[state.op](state)


# ------------------------------------------------------------------ in 64 bits


def _exact_tree(s):
    md = s.md
    hkv = s.cache.shape[3]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    group = s.q.shape[1] // hkv
    mask = md.tree_mask.cpu().numpy().astype(np.uint64)
    for i, (c, n) in enumerate(zip(md.context_lens_cpu, md.seq_lens_cpu)):
        a, b = md.query_start_loc_cpu[i:i + 2]
        pages = md.block_tables[i, :-(-n // PAGE)].long()
        keys = s.cache[0][pages].reshape(-1, hkv, s.q.shape[2])[:n].double()
        vals = s.cache[1][pages].reshape(-1, hkv, s.q.shape[2])[:n].double()
        drafted = np.array([[(int(mask[r, x // WORD]) >> (x % WORD)) & 1 for x in range(b - a)] for r in range(a, b)], dtype=bool)
        hidden = torch.zeros(b - a, n, dtype=torch.bool, device=DEV)
        hidden[:, c:] = torch.from_numpy(~drafted).to(DEV)
        for h in range(s.q.shape[1]):
            w = s.q[a:b, h].double() @ keys[:, h // group].T.contiguous() * s.scale
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[a:b, h] = w @ vals[:, h // group].contiguous()
    return out


def _exact_commit(s):
    md = s.md
    parents, draft, target = s.parents.tolist(), s.draft.tolist(), s.target.tolist()
    tables = md.block_tables.tolist()
    stack = s.stack.double()
    for i, c in enumerate(md.context_lens_cpu):
        a, b = md.query_start_loc_cpu[i:i + 2]
        cur, path = 0, [0]
        while True:
            hits = [x for x in range(b - a) if parents[a + x] == cur and draft[a + x] == target[a + cur]]
            if not hits:
                break
            cur = hits[0]
            path.append(cur)
        where = [(tables[i][(c + x) // PAGE], (c + x) % PAGE) for x in range(b - a)]
        for to, x in enumerate(path):
            stack[:, :, where[to][0], where[to][1]] = stack[:, :, where[x][0], where[x][1]].clone()
    return None, None, None, stack


def _exact_select(s):
    x = s.logits.float().cpu().numpy().astype(np.float64)
    base = s.scores.cpu().numpy().astype(np.float64)
    top = x.max(1, keepdims=True)
    total = base[:, None] + (x - (top + np.log(np.exp(x - top).sum(1, keepdims=True))))
    total = total.reshape(-1, s.beams * x.shape[1])
    return np.stack([np.sort(np.partition(r, len(r) - s.n)[len(r) - s.n:])[::-1] for r in total]), None, None


def _exact_reorder(s):
    groups, k = s.beams.shape
    tables, lens, beams = s.tables.tolist(), s.lens.tolist(), s.beams.tolist()
    stack = s.stack.double()
    for g in range(groups):
        n = lens[g * k]
        page = [tables[g * k + b][n // PAGE] for b in range(k)]
        old = [stack[:, :, p, :n % PAGE].clone() for p in page]
        for b in range(k):
            stack[:, :, page[b], :n % PAGE] = old[beams[g][b]]
    return None, stack


def exact(case, seed):
    return {"tree": _exact_tree, "commit": _exact_commit, "select": _exact_select,
            "reorder": _exact_reorder}[case["op"]](prepare(case, seed))
