"""A windowed step as it is used: lengths and pages in, attention out, and a model of windows and head norms through
LLM.generate, against plain implementations.

The model's tolerances are those of ``test_generate_gpu`` (2 layers of hidden 256, a bf16 model against fp32): the step is
the same but for which keys the rows see and one rounding of q and k less.
"""

import random

import pytest
import torch

from babyvllm.kernels.qk_norm_rope import fused_qk_norm_rope_and_cache
from babyvllm.kernels.step_tables import build_step_tables
from babyvllm.kernels.window_attn import paged_window_attention
from babyvllm.worker.context import AttentionMetadata, set_forward_context
from tests import _generate as G
from tests.test_generate_gpu import LOGIT_MAX_TOL, LOGIT_MEAN_TOL, LOGIT_TOL, NEW_TOKENS
from tests.test_qk_norm_rope_gpu import near, rotated
from tests.test_step_tables_gpu import formula as tables_formula, held_entries
from tests.test_window_attn_gpu import check, formula

pytestmark = pytest.mark.gpu
PAGE = 16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Chat:
    """Sequences over one cache that give back the pages their rows no longer see."""

    def __init__(self, seqs, heads, hkv, d, window, sinks, pages=200):
        g = torch.Generator(device="cuda").manual_seed(0)
        self.heads, self.hkv, self.d, self.window, self.sinks = heads, hkv, d, window, sinks
        self.cache = torch.full((2, pages, PAGE, hkv, d), float("nan"), device="cuda", dtype=torch.bfloat16)
        self.free = list(range(pages))
        random.Random(0).shuffle(self.free)
        self.held = [{} for _ in range(seqs)]  # entry -> page
        self.ctx = [0] * seqs
        self.keys = [torch.zeros(0, hkv, d, device="cuda") for _ in range(seqs)]
        self.vals = [torch.zeros(0, hkv, d, device="cuda") for _ in range(seqs)]
        self.w = [(1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2)]
        self.gen = g

    def step(self, new):
        for s, n in enumerate(new):
            want = held_entries(self.ctx[s], n, self.window, self.sinks)
            for i in [i for i in self.held[s] if i not in want]:
                page = self.held[s].pop(i)
                self.cache[:, page] = float("nan")  # as another request's would be
                self.free.insert(0, page)
            for i in want:
                if i not in self.held[s]:
                    self.held[s][i] = self.free.pop()
        listed = [h[i] for h in self.held for i in sorted(h)]
        rows, width = sum(new), 40
        t = build_step_tables(i32(new), i32(self.ctx), i32(listed), rows + 3, width, window=self.window, sinks=self.sinks)
        want = tables_formula(new, self.ctx, listed, rows + 3, width, self.window, self.sinks)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(t, want))
        qkv = torch.randn(rows + 3, self.heads + 2 * self.hkv, self.d, device="cuda", generator=self.gen).to(torch.bfloat16)
        q, k, v = qkv.split([self.heads, self.hkv, self.hkv], dim=1)
        angle = t.positions.double()[:, None] * torch.logspace(0, -3, self.d // 2, device="cuda", dtype=torch.float64).repeat(2)
        cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
        turned = fused_qk_norm_rope_and_cache(q, k, v, *self.w, 1e-6, cos, sin, self.cache, t.slot_mapping)
        near(turned, rotated(q, self.w[0], 1e-6, cos, sin), "q")
        qsl = t.query_start_loc.tolist()
        ctx = i32(self.ctx)
        md = AttentionMetadata(t.slot_mapping, t.block_tables, t.query_start_loc, t.seq_lens, ctx, qsl, t.seq_lens.tolist(),
                               list(self.ctx), max(new), max(t.seq_lens.tolist()))
        out = paged_window_attention(turned, self.cache, md, 0.125, self.window, self.sinks)
        check(out, formula(turned, self.cache, md, 0.125, self.window, self.sinks))
        # The cache holds what the step appended: every key that the rows see, from the start of the sequence on.
        kk, _ = rotated(k, self.w[1], 1e-6, cos, sin)
        for s, n in enumerate(new):
            self.keys[s] = torch.cat((self.keys[s], kk[qsl[s]:qsl[s + 1]].float()))
            self.vals[s] = torch.cat((self.vals[s], v[qsl[s]:qsl[s + 1]].float()))
            self.ctx[s] += n
            for r in range(qsl[s], qsl[s + 1]):
                p = self.ctx[s] - n + r - qsl[s]
                sees = [j for j in range(p + 1) if j > p - self.window or j < self.sinks]
                group = self.heads // self.hkv
                key, val = (x[s][sees].repeat_interleave(group, 1) for x in (self.keys, self.vals))
                w = torch.softmax((key * turned[r].float()).sum(-1) * 0.125, 0)
                o = (w[..., None] * val).sum(0)
                # bf16 keys: each score off by 2^-8 of |q||k| / 8 at most; 2^-8 of the weights and of the output.
                reach = (w[..., None] * (val - o).abs()).sum(0)
                slack = 2 ** -8 * 0.125 * (key.norm(dim=-1) * turned[r].float().norm(dim=-1)).amax(0)[..., None]
                tol = (torch.exp(2 * slack) - 1 + 2 ** -7) * reach + 2 ** -7 * (w[..., None] * val.abs()).sum(0) + 1e-6
                assert ((out[r].float() - o).abs() <= tol).all()


@pytest.mark.parametrize("heads,hkv,d", [(14, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(40, 4), (33, 0), (64, 20)])
def test_prompts_and_decode_steps_over_a_cache_that_gives_pages_back(heads, hkv, d, window, sinks):
    chat = Chat(4, heads, hkv, d, window, sinks)
    chat.step([70, 1, 33, 0])
    for _ in range(3):
        chat.step([1, 1, 1, 1])
    chat.step([1, 90, 0, 40])
    chat.step([30, 1, 1, 1])
    for _ in range(4):
        chat.step([1, 1, 1, 1])


def config(**k):
    from babyvllm.config import ModelConfig
    return ModelConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                       num_attention_heads=4, num_key_value_heads=2, rms_norm_eps=1e-6,
                       max_position_embeddings=4096, rope_theta=10000.0, tie_word_embeddings=False, **k)


def llm_of(cfg, graphs=True, blocks=256):
    from babyvllm.config import CacheConfig, SchedulerConfig
    from babyvllm.llm import LLM
    llm = LLM(cfg, cache_config=CacheConfig(num_gpu_blocks=blocks), scheduler_config=SchedulerConfig(
        max_num_seqs=8, max_num_batched_tokens=160), use_cuda_graphs=graphs, seed=3, init_std=0.1)
    if cfg.qk_norm:  # weights that are not all 1
        g = torch.Generator(device="cuda").manual_seed(9)
        for layer in llm.model_runner.model.model.layers:
            for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                norm.weight.data.copy_(1 + 0.2 * torch.randn(64, device="cuda", generator=g))
    return llm


@torch.no_grad()
def plain_logits(model, cfg, ids):
    """The model of `cfg` in fp32, a whole sequence at once."""
    w = {k: v.float() for k, v in model.state_dict().items()}
    norm = lambda x, name: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.rms_norm_eps) * w[name]  # noqa: E731
    n, d, h, hkv = len(ids), cfg.head_dim, cfg.num_attention_heads, cfg.num_key_value_heads
    pos = torch.arange(n, device="cuda")
    angle = pos.double()[:, None] * cfg.rope_theta ** (-torch.arange(0, d, 2, device="cuda").double() / d)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turn = lambda x: torch.cat((x[..., :d // 2] * cos - x[..., d // 2:] * sin,  # noqa: E731
                                x[..., d // 2:] * cos + x[..., :d // 2] * sin), -1)
    i, j = pos[:, None], pos[None]
    seen = j <= i
    if cfg.sliding_window is not None:
        seen &= (j > i - cfg.sliding_window) | (j < cfg.attention_sinks)
    x = w["model.embed_tokens.weight"][torch.tensor(ids, device="cuda")]
    for layer in range(cfg.num_hidden_layers):
        p = f"model.layers.{layer}."
        y = norm(x, p + "input_layernorm.weight") @ w[p + "self_attn.qkv_proj.weight"].T + w[p + "self_attn.qkv_proj.bias"]
        q, k, v = (t.view(n, -1, d) for t in y.split([h * d, hkv * d, hkv * d], -1))
        if cfg.qk_norm:
            q, k = norm(q, p + "self_attn.q_norm.weight"), norm(k, p + "self_attn.k_norm.weight")
        q, k, v = turn(q), turn(k).repeat_interleave(h // hkv, 1), v.repeat_interleave(h // hkv, 1)
        heads = []
        for a in range(h):
            score = (q[:, a] @ k[:, a].T / d ** 0.5).masked_fill(~seen, float("-inf"))
            heads.append(torch.softmax(score, -1) @ v[:, a])
        x = x + torch.cat(heads, -1) @ w[p + "self_attn.o_proj.weight"].T
        y = norm(x, p + "post_attention_layernorm.weight") @ w[p + "mlp.gate_up_proj.weight"].T
        gate, up = y.chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w[p + "mlp.down_proj.weight"].T
    return norm(x, "model.norm.weight") @ w["lm_head.weight"].T


def prompts():
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 512, (n,), generator=g).tolist() for n in (5, 17, 40, 150, 3, 90)]


@pytest.mark.parametrize("options", [dict(sliding_window=24, attention_sinks=4), dict(qk_norm=True),
                                     dict(sliding_window=33, attention_sinks=0, qk_norm=True)], ids=str)
def test_generation_against_a_plain_model(options):
    cfg = config(**options)
    llm = llm_of(cfg)
    toks, logits = G.generate_recording(llm, prompts(), NEW_TOKENS)
    assert llm.model_runner.graph_replays > 0
    want = [plain_logits(llm.model_runner.model, cfg, p + t[:-1])[len(p) - 1:].cpu() for p, t in zip(prompts(), toks)]
    exact, total, worst_max, worst_mean = G.compare_with_checker(toks, logits, want, LOGIT_MAX_TOL, LOGIT_MEAN_TOL)
    print(options, exact, total, worst_max, worst_mean)
    assert exact >= 0.9 * total
    other, _ = G.generate_recording(llm_of(cfg, graphs=False), prompts(), NEW_TOKENS)
    for a, b, x in zip(toks, other, want):
        clear = G.clear_prefix(x, LOGIT_TOL)
        assert a[:clear] == b[:clear]


def test_norm_modules_with_hooks_are_called():
    cfg = config(qk_norm=True)
    plain, hooked = llm_of(cfg, graphs=False), llm_of(cfg, graphs=False)
    seen = []
    for layer in hooked.model_runner.model.model.layers:
        layer.self_attn.k_norm.register_forward_hook(lambda m, a, out: seen.append(out[0].shape))
    _, a = G.generate_recording(plain, prompts(), 4)
    _, b = G.generate_recording(hooked, prompts(), 4)
    assert seen and all(s[1:] == (2, 64) for s in seen)
    # (Three roundings of q and k more: of the normed value, of both products of the rotation.)
    assert max((x[0] - y[0]).abs().max().item() for x, y in zip(a, b)) <= LOGIT_MAX_TOL


def test_a_window_of_everything_is_no_window():
    full, wide = llm_of(config()), llm_of(config(sliding_window=4096))
    _, a = G.generate_recording(full, prompts(), 4)
    _, b = G.generate_recording(wide, prompts(), 4)
    assert max((x[0] - y[0]).abs().max().item() for x, y in zip(a, b)) <= LOGIT_TOL


def test_the_runner_gives_the_kernels_what_its_host_path_does():
    llm = llm_of(config(), graphs=False)
    runner, seen = llm.model_runner, []
    inner = runner.prepare_inputs

    def both(out):
        got = inner(out)
        runner.block_size = 0  # the host path
        want = inner(out)
        runner.block_size = 16
        seen.append(len(out.scheduled_sequences))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for name in ("slot_mapping", "query_start_loc", "seq_lens", "context_lens"):
            x, y = getattr(got[2], name), getattr(want[2], name)
            assert x.dtype == y.dtype and torch.equal(x, y), name
        for s, n in enumerate(want[2].seq_lens_cpu):
            assert torch.equal(got[2].block_tables[s, :-(-n // 16)], want[2].block_tables[s, :-(-n // 16)])
        assert got[2].block_tables.shape == want[2].block_tables.shape
        return got

    runner.prepare_inputs = both
    G.generate_recording(llm, prompts(), 5)
    assert max(seen) > 1 and len(seen) > 5


def test_trees_are_refused_by_a_layer_with_a_window():
    from babyvllm.layers.attention import Attention
    with pytest.raises(ValueError, match="window"):
        Attention(2, 64, 1, window=0)
    layer = Attention(2, 64, 1, window=8)
    layer.kv_cache = torch.zeros(2, 4, PAGE, 1, 64, device="cuda", dtype=torch.bfloat16)
    one = i32([1])
    md = AttentionMetadata(None, i32([[0]]), i32([0, 1]), one, one, [0, 1], [1], [1], 1, 1, tree_mask=torch.ones(1, 1, device="cuda"))
    q = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    with set_forward_context(md), pytest.raises(RuntimeError, match="window"):
        layer(q, q[:, :1], q[:, :1])
