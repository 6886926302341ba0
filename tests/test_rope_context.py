"""Rotary tables reach as far as the positions go: scaled contexts, sequences and engines beyond a model's context."""
import pytest
import torch

from skyrl_b200.engine.llm_engine import EngineConfig, LLMEngine, SamplingParams
from skyrl_b200.models.decoder import CausalLM, ModelArgs

KINDS = {"whole": {}, "part": dict(partial_rotary_factor=0.5), "norms": dict(qk_norm=True)}


def model(context, kind="whole", device="cpu", **kw):
    D = 64 if device == "cpu" else 128  # the attention kernels' head size
    a = ModelArgs(vocab_size=96, hidden_size=4 * D, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=D, intermediate_size=256,
                  tie_word_embeddings=True, max_position_embeddings=context, **KINDS[kind], **kw)
    return CausalLM(a, device=device, dtype=torch.float32 if device == "cpu" else torch.bfloat16, seed=11)


def hidden(m, n, device="cpu"):
    ids = torch.arange(n, device=device) * 7 % 90
    with torch.no_grad():
        return m(ids, torch.arange(n, device=device, dtype=torch.int32), torch.tensor([0, n], device=device, dtype=torch.int32), n)


def beyond_the_context(kind, device):
    want = hidden(model(512, kind, device), 100, device)
    got = hidden(model(32, kind, device), 100, device)
    assert torch.isfinite(want).all() and torch.equal(got, want)


def engine_beyond_the_context(kind, device):
    cfg = EngineConfig(block_size=16 if device == "cuda" else 4, max_num_seqs=2, max_model_len=96, num_blocks=64, enforce_eager=True)
    sp = SamplingParams(max_tokens=50, temperature=0.0, ignore_eos=True)
    outs = [LLMEngine(model(c, kind, device), cfg).generate([[5, 6, 7]], sp)[0] for c in (32, 512)]
    assert outs[0].token_ids == outs[1].token_ids and outs[0].logprobs == outs[1].logprobs


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_sequence(kind):
    beyond_the_context(kind, "cpu")


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_engine(kind):
    engine_beyond_the_context(kind, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_sequence_and_engine_on_the_gpu(kind):
    beyond_the_context(kind, "cuda")
    engine_beyond_the_context(kind, "cuda")


@pytest.mark.parametrize("scaling,rows", [
    ({"rope_type": "linear", "factor": 2.0}, 128),
    ({"type": "linear", "factor": 4}, 256),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}, 128),
    ({"rope_type": "default"}, 64),
    (None, 64),
])
def test_rows_of_scaled_contexts(scaling, rows):
    assert model(64, rope_scaling=scaling).rope_table("cpu").shape == (rows, 64)


def test_a_longer_table_leaves_the_one_before_it_alone():
    m = model(64)
    first = m.rope_table("cpu")
    copy = first.clone()
    assert m.rope_table("cpu", 64) is first and m.rope_table("cpu") is first
    second = m.rope_table("cpu", 65)
    assert second.shape[0] == 128 and torch.equal(second[:64], first)
    assert m.rope_table("cpu", 128) is second and m.rope_table("cpu") is second
    assert m.rope_table("cpu", 1000).shape[0] == 1000
    assert torch.equal(first, copy) and any(t is first for t in m._rope_tables_before)
