"""Decoding with several candidates of a request, whole: the model, the paged cache and the kernels together.

Both tests run a small random Qwen2 (2 layers, hidden 256, 4 / 2 heads of 64, vocabulary 512)
and compare every logits row with the same model's row for the same tokens, computed
without candidates. Each of the two is within 0.2 (0.06 on average) of the exact model by the
bounds of the end-to-end generation tests, which run this model, so they are within
twice that of each other. A token that attends another branch, or a row moved to a wrong
place, changes logits (about N(0, 1.6^2)) by their own size.
"""

import random

import pytest
import torch

from babyvllm.config import ModelConfig
from babyvllm.kernels.argmax import greedy_argmax
from babyvllm.kernels.beam import beam_select, reorder_beams
from babyvllm.kernels.tree_attn import ancestor_masks
from babyvllm.kernels.tree_commit import commit_draft_tree
from babyvllm.models.qwen2 import Qwen2ForCausalLM
from babyvllm.worker.context import AttentionMetadata, set_forward_context

pytestmark = pytest.mark.gpu
PAGE, VOCAB = 16, 512
LOGIT_MAX_TOL = 2 * 0.2
LOGIT_MEAN_TOL = 2 * 0.06


class Served:
    """The model with a paged cache; a step takes each row's tokens behind its context."""

    def __init__(self, num_pages):
        cfg = ModelConfig(vocab_size=VOCAB, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                          num_attention_heads=4, num_key_value_heads=2, rms_norm_eps=1e-6,
                          max_position_embeddings=4096, rope_theta=10000.0, tie_word_embeddings=False)
        with torch.device("cuda"):
            self.model = Qwen2ForCausalLM(cfg).to(torch.bfloat16).eval()
        self.model.init_random(3, 0.1)
        self.caches = []
        for layer in self.model.model.layers:
            # Unwritten slots hold NaN: nothing may read them.
            cache = torch.full((2, num_pages, PAGE, cfg.num_key_value_heads, cfg.head_dim), float("nan"),
                               device="cuda", dtype=torch.bfloat16)
            layer.self_attn.attn.kv_cache = cache
            self.caches.append(cache)

    @torch.no_grad()
    def step(self, tokens, contexts, tables, depths=None, tree_mask=None):
        """Logits of every row (fp32) and the step's metadata."""
        qsl = [0]
        for t in tokens:
            qsl.append(qsl[-1] + len(t))
        slots = [tables[s][p // PAGE] * PAGE + p % PAGE
                 for s, t in enumerate(tokens) for p in range(contexts[s], contexts[s] + len(t))]
        positions = [contexts[s] + (depths[qsl[s] + i] if depths is not None else i)
                     for s, t in enumerate(tokens) for i in range(len(t))]
        lens = [c + len(t) for c, t in zip(contexts, tokens)]
        i32 = dict(dtype=torch.int32, device="cuda")
        md = AttentionMetadata(
            slot_mapping=torch.tensor(slots, device="cuda"), block_tables=torch.tensor(tables, **i32),
            query_start_loc=torch.tensor(qsl, **i32), seq_lens=torch.tensor(lens, **i32),
            context_lens=torch.tensor(contexts, **i32), query_start_loc_cpu=qsl, seq_lens_cpu=lens,
            context_lens_cpu=list(contexts), max_query_len=max(map(len, tokens)), max_seq_len=max(lens),
            tree_mask=None if tree_mask is None else tree_mask.cuda())
        ids = torch.tensor([x for t in tokens for x in t], device="cuda")
        with set_forward_context(md):
            hidden = self.model(ids, torch.tensor(positions, device="cuda"))
        return self.model.compute_logits(hidden), md


def fresh_tables(rows, width, first=0):
    """Shuffled tables of pages of their own."""
    order = list(range(first, first + rows * width))
    random.Random(rows * width).shuffle(order)
    return [order[i * width:(i + 1) * width] for i in range(rows)]


def assert_logits_close(got, want):
    diff = (got.float() - want.float()).abs()
    assert diff.max() <= LOGIT_MAX_TOL and diff.mean() <= LOGIT_MEAN_TOL, (diff.max(), diff.mean())


def drafted_tree(rng, following, longest):
    """Tokens, parents and the path of the right ones: a path of `following`'s tokens, among wrong branches."""
    depth = rng.randint(0, min(longest, len(following) - 1))
    tokens, parents, path = [following[0]], [-1], [0]
    for i in range(1, depth + 1):
        for _ in range(rng.randint(0, 2)):  # a wrong branch from anywhere, before the right child
            parents.append(rng.randrange(len(tokens)))
            # (Of equal siblings the first counts: one before the right child has another token.)
            tokens.append((following[i] + 1 + rng.randrange(VOCAB - 1)) % VOCAB)
        parents.append(path[-1])
        tokens.append(following[i])
        path.append(len(tokens) - 1)
    for _ in range(rng.randint(0, 3)):
        parents.append(rng.randrange(len(tokens)))
        tokens.append(rng.randrange(VOCAB))
    return tokens, parents, path


def test_verified_trees_continue_like_one_token_at_a_time():
    prompts_rng, new = random.Random(11), 40
    lengths = [5, 16, 61, 130, 333]
    prompts = [[prompts_rng.randrange(VOCAB) for _ in range(n)] for n in lengths]
    width = (max(lengths) + new + 40) // PAGE + 2
    served = Served(2 * len(prompts) * width)
    one, drafted = fresh_tables(len(prompts), width), fresh_tables(len(prompts), width, len(prompts) * width)

    # One token at a time.
    last = [sum(lengths[:i + 1]) - 1 for i in range(len(lengths))]
    logits, _ = served.step(prompts, [0] * len(prompts), one)
    sequential = [logits[last].float()]
    chosen = [[t] for t in sequential[0].argmax(-1).tolist()]
    for i in range(new):
        logits, _ = served.step([[c[-1]] for c in chosen], [n + i for n in lengths], one)
        sequential.append(logits.float())
        for c, t in zip(chosen, sequential[-1].argmax(-1).tolist()):
            c.append(t)

    # Drafted trees: from the same tokens and wrong ones. `done`: tokens of `chosen` that are in
    # the cache behind the prompt.
    served.step(prompts, [0] * len(prompts), drafted)
    rng, done, accepted_lengths = random.Random(5), [0] * len(prompts), []
    while min(done) + 8 < new:
        trees = [drafted_tree(rng, c[n:min(n + 8, new)], 6) for c, n in zip(chosen, done)]
        masks, depths = ancestor_masks([t[1] for t in trees])
        contexts = [n + k for n, k in zip(lengths, done)]
        logits, md = served.step([t[0] for t in trees], contexts, drafted, depths.tolist(), masks)
        answers = torch.empty(logits.shape[0], device="cuda", dtype=torch.int64)
        greedy_argmax(logits, answers)
        logits = logits.float()
        for s, (tokens, _, path) in enumerate(trees):
            for depth, node in enumerate(path):
                row = logits[md.query_start_loc_cpu[s] + node]
                want = sequential[done[s] + depth + 1][s]
                assert_logits_close(row, want)
                # (Near-ties may fall otherwise: the comparison goes on with the tokens from above.)
                answers[md.query_start_loc_cpu[s] + node] = chosen[s][done[s] + depth + 1]
        flat = torch.tensor([x for t in trees for x in t[0]], device="cuda")
        parents = torch.tensor([x for t in trees for x in t[1]], device="cuda", dtype=torch.int32)
        path, accepted, following = commit_draft_tree(served.caches, md, flat, answers, parents)
        for s, (tokens, par, want) in enumerate(trees):
            n = int(accepted[s])
            got = path[s, :n].tolist()
            assert got[:len(want)] == want and (path[s, n:] == -1).all()
            # A wrong node behind the path's end may hold the right token by chance.
            assert [tokens[i] for i in got] == chosen[s][done[s]:done[s] + n]
            assert int(following[s]) == chosen[s][done[s] + n] or n > len(want)
            accepted_lengths.append(n)
            done[s] += n
        done = [min(d, new - 1) for d in done]
    assert max(accepted_lengths) >= 5 and min(accepted_lengths) == 1
    # What the cache holds of the accepted tokens is what one token at a time left there (up to
    # ten bf16 roundings of 2^-9 rms each, in each of the two).
    for cache in served.caches:
        for s, n in enumerate(lengths):
            for p in range(n + done[s]):
                a = cache[:, one[s][p // PAGE], p % PAGE].float()
                b = cache[:, drafted[s][p // PAGE], p % PAGE].float()
                assert (a - b).norm() <= 0.02 * a.norm()


def test_beams_continue_like_their_own_prompts():
    rng, k, new = random.Random(3), 4, 20
    lengths = [37, 5, 112]
    prompts = [[rng.randrange(VOCAB) for _ in range(n)] for n in lengths]
    groups, rows = len(prompts), len(prompts) * k
    width = (max(lengths) + new) // PAGE + 2
    served = Served(2 * rows * width + groups * width)
    own = fresh_tables(rows, width)                    # page i of a row's own, for the i-th page it fills
    again = fresh_tables(rows, width, rows * width)    # for the recomputation
    # The prompts run once, in the first beam's pages; every beam starts from them.
    logits, _ = served.step(prompts, [0] * groups, [own[g * k] for g in range(groups)])
    last = [sum(lengths[:g + 1]) - 1 for g in range(groups)]
    logits = logits[last].repeat_interleave(k, 0)
    tables = torch.tensor(own, dtype=torch.int32, device="cuda")
    lens = [n for n in lengths for _ in range(k)]
    reorder_beams(served.caches, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                  torch.zeros(groups, k, dtype=torch.int64, device="cuda"))
    scores = torch.full((groups, k), -float("inf"), device="cuda")
    scores[:, 0] = 0.0                                 # the first step: one beam, k continuations
    texts = [list(prompts[g]) for g in range(groups) for _ in range(k)]
    forked = 0
    for i in range(new):
        totals = (scores.reshape(-1, 1).double() + torch.log_softmax(logits.double(), -1)).view(groups, -1)
        scores, beams, tokens = beam_select(logits, scores, k, k)
        assert torch.allclose(scores.double(), totals.topk(k).values, rtol=2 ** -24, atol=2 ** -18)
        parents = beams.tolist()
        if i > 0:
            reorder_beams(served.caches, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), beams)
        forked += sum(len(set(p)) < k for p in parents)
        texts = [texts[g * k + parents[g][b]] + [int(tokens[g, b])] for g in range(groups) for b in range(k)]
        logits, _ = served.step([t[-1:] for t in texts], lens, tables.tolist())
        lens = [n + 1 for n in lens]
        # A row's next page is its own again: full pages behind it are shared.
        for row, n in enumerate(lens):
            assert int(tables[row, n // PAGE]) == own[row][n // PAGE]
        # The same texts from scratch.
        full, md = served.step(texts, [0] * rows, again)
        want = full[[q - 1 for q in md.query_start_loc_cpu[1:]]]
        assert_logits_close(logits, want)
        # Scores are the texts' log-probabilities.
        logp = torch.log_softmax(full.float(), -1)
        for row, text in enumerate(texts):
            g, start = row // k, md.query_start_loc_cpu[row]
            rest = range(lengths[g], len(text))
            total = sum(float(logp[start + p - 1, text[p]]) for p in rest)
            assert abs(float(scores[g, row % k]) - total) <= len(rest) * 2 * LOGIT_MAX_TOL
        assert (scores[:, :-1] >= scores[:, 1:]).all()
        assert len({tuple(t) for t in texts}) == rows
    assert forked >= groups
