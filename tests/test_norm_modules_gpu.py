"""Head norms of other classes than the framework's: a module may return the normed tensor, or a tuple that starts with it."""

import pytest
import torch

from tests import _generate as G
from tests.test_generate_gpu import LOGIT_MAX_TOL
from tests.test_windowed_model_gpu import config, llm_of, prompts

pytestmark = pytest.mark.gpu


class Paired(torch.nn.Module):
    """x · rsqrt(mean(x²) + eps) · weight in fp32, returned as (normed, x)."""

    def __init__(self, weight, eps, pair):
        super().__init__()
        self.weight, self.eps, self.pair = weight, eps, pair

    def forward(self, x):
        y = x.float()
        y = (y * torch.rsqrt((y * y).mean(-1, keepdim=True) + self.eps) * self.weight.float()).to(x.dtype)
        return [y, x] if self.pair == "list" else (y, x) if self.pair else y


def torch_norm(old):
    new = torch.nn.RMSNorm(64, eps=old.eps, device="cuda", dtype=torch.bfloat16)
    new.weight = old.weight
    return new


KINDS = {
    "torch": torch_norm,
    "tensor": lambda old: Paired(old.weight, old.eps, False),
    "tuple": lambda old: Paired(old.weight, old.eps, True),
    "list": lambda old: Paired(old.weight, old.eps, "list"),
}


@pytest.mark.parametrize("which", [("q_norm", "k_norm"), ("k_norm",)], ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_norms_of_another_class(kind, which):
    cfg = config(qk_norm=True)
    plain, other = llm_of(cfg, graphs=False), llm_of(cfg, graphs=False)
    for layer in other.model_runner.model.model.layers:
        for name in which:
            setattr(layer.self_attn, name, KINDS[kind](getattr(layer.self_attn, name)))
    _, a = G.generate_recording(plain, prompts(), 4)
    _, b = G.generate_recording(other, prompts(), 4)
    # (Roundings of q and k more than the fused form's: of the normed value, of both products of the rotation.)
    assert max((x[0] - y[0]).abs().max().item() for x, y in zip(a, b)) <= LOGIT_MAX_TOL


def test_a_hook_that_returns_a_tensor():
    cfg = config(qk_norm=True)
    plain, hooked = llm_of(cfg, graphs=False), llm_of(cfg, graphs=False)
    for layer in hooked.model_runner.model.model.layers:
        layer.self_attn.q_norm.register_forward_hook(lambda m, a, out: out[0])
    _, a = G.generate_recording(plain, prompts(), 4)
    _, b = G.generate_recording(hooked, prompts(), 4)
    assert max((x[0] - y[0]).abs().max().item() for x, y in zip(a, b)) <= LOGIT_MAX_TOL
