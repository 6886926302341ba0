"""Log-probabilities of a small batch of an expert model, with and without gradients: one computation."""
import dataclasses

import pytest
import torch

from skyrl_b200.models import moe
from skyrl_b200.models.decoder import PRESETS, CausalLM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 9, 30])
def test_scores_are_those_of_the_training_forward(n):
    m = CausalLM(dataclasses.replace(PRESETS["tiny-moe"], num_layers=3), device="cuda", dtype=torch.bfloat16, seed=5)
    g = torch.Generator().manual_seed(n)
    ids, tgt = (torch.randint(0, m.args.vocab_size, (n,), generator=g).cuda() for _ in range(2))
    pos, cu = torch.arange(n, device="cuda", dtype=torch.int32), torch.tensor([0, n], device="cuda", dtype=torch.int32)

    def scores():
        h = m(ids, pos, cu, n)
        return h.detach(), m.token_logprobs(h, tgt)[0].detach()

    with torch.no_grad():
        h = m._p["embed"][ids]
        pre = "layers.0."
        assert moe._takes_few(h, *(m.p(pre + w) for w in ("router", "experts_wgu", "experts_wd")), m.args.num_experts_per_tok)
        scored = scores()
    for a, b in zip(scored, scores()):
        assert torch.equal(a, b)
