"""Which forwards of an expert model may take the layer for a few tokens: the engine's, not those that score tokens."""
import dataclasses

import pytest
import torch

from skyrl_b200.engine.llm_engine import EngineConfig, LLMEngine, SamplingParams
from skyrl_b200.models import moe
from skyrl_b200.models.decoder import PRESETS, CausalLM


@pytest.fixture
def calls(monkeypatch):
    seen, real = [], moe.moe_ffn

    def spy(*a, **kw):
        seen.append((kw.get("few_tokens", True), torch.is_grad_enabled()))
        return real(*a, **kw)

    monkeypatch.setattr(moe, "moe_ffn", spy)
    return seen


def test_only_the_engine_takes_the_path_for_few_tokens(calls):
    a = dataclasses.replace(PRESETS["tiny-moe"], num_layers=2)
    m = CausalLM(a, dtype=torch.float32, seed=3)
    ids, cu = torch.arange(4, 15), torch.tensor([0, 11], dtype=torch.int32)
    pos = torch.arange(11, dtype=torch.int32)
    with torch.no_grad():
        m(ids, pos, cu, 11)
    m(ids, pos, cu, 11)
    assert calls == [(False, False)] * 2 + [(False, True)] * 2
    calls.clear()
    LLMEngine(m, EngineConfig(block_size=4, max_num_seqs=2, max_model_len=32, enforce_eager=True)).generate(
        [ids.tolist()], SamplingParams(max_tokens=2, temperature=0.0, ignore_eos=True))
    assert calls and all(c == (True, False) for c in calls)
