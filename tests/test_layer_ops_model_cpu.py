"""Rotary variants, head norms, cache rows, paged layout and experts together, as models and the engine use them."""
import pytest
import torch

from skyrl_b200.engine.llm_engine import EngineConfig, LLMEngine, SamplingParams
from skyrl_b200.models import hf_io
from skyrl_b200.models.decoder import CausalLM, ModelArgs

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 64}
KINDS = {
    "norms": dict(qk_norm=True, rope_scaling=YARN),
    "neighbours": dict(rope_interleaved=True, partial_rotary_factor=0.5),
    "norms-part": dict(qk_norm=True, partial_rotary_factor=0.5, rope_scaling={"type": "linear", "factor": 2.0}),
    "experts": dict(qk_norm=True, rope_scaling=LLAMA3, num_experts=6, num_experts_per_tok=2, moe_intermediate_size=24),
}


def model(kind, **kw):
    args = ModelArgs(vocab_size=97, hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16,
                     intermediate_size=96, tie_word_embeddings=True, max_position_embeddings=256, **KINDS[kind])
    m = CausalLM(args, dtype=torch.float32, seed=11, **kw)
    with torch.no_grad():
        for name, p in m.named_flat_views():
            if name.endswith(("q_norm", "k_norm")):
                p.copy_(1 + 0.3 * torch.randn(p.shape, generator=torch.Generator().manual_seed(len(name))))
    return m


def greedy(m, prompt, n):
    toks = list(prompt)
    for _ in range(n):
        ids = torch.tensor(toks)
        with torch.no_grad():
            z = m.logits(m(ids, torch.arange(len(toks), dtype=torch.int32), torch.tensor([0, len(toks)], dtype=torch.int32), len(toks)))
        toks.append(int(z[-1].argmax()))
    return toks[len(prompt):]


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_engine_decodes_what_the_full_forward_gives(kind):
    m = model(kind)
    eng = LLMEngine(m, EngineConfig(block_size=4, max_num_seqs=3, max_model_len=64, max_num_batched_tokens=64, sync_interval=3,
                                    enforce_eager=True))
    prompts = [[5, 6, 7, 8, 9], [10, 11], [3] * 9, [20, 21, 22], [40]]
    for p, o in zip(prompts, eng.generate(prompts, SamplingParams(max_tokens=7, temperature=0.0))):
        assert o.token_ids == greedy(m, p, 7)


def test_prefix_cache_and_routing_capture():
    m = model("experts")
    shared = list(range(2, 20))
    prompts = [shared + [30 + i] for i in range(4)]
    want = [greedy(m, p, 5) for p in prompts]
    eng = LLMEngine(m, EngineConfig(block_size=4, max_num_seqs=4, max_model_len=64, enable_prefix_caching=True, enforce_eager=True))
    first = eng.generate(prompts[:1], SamplingParams(max_tokens=5, temperature=0.0))
    rest = eng.generate(prompts[1:], SamplingParams(max_tokens=5, temperature=0.0))
    assert [o.token_ids for o in first + rest] == want and eng.stats.get("prefix_cached_tokens", 0) > 0
    eng = LLMEngine(m, EngineConfig(block_size=4, max_num_seqs=4, max_model_len=64, enforce_eager=True, return_routed_experts=True))
    for o, w in zip(eng.generate(prompts, SamplingParams(max_tokens=5, temperature=0.0)), want):
        assert o.token_ids == w and int(o.routed_experts.min()) >= 0 and int(o.routed_experts.max()) < 6


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_training_gradients_accumulate_and_survive_checkpointing(kind):
    ids = torch.randint(0, 97, (23,), generator=torch.Generator().manual_seed(1))
    pos = torch.cat([torch.arange(9), torch.arange(14)]).to(torch.int32)
    cu, tgt = torch.tensor([0, 9, 23], dtype=torch.int32), torch.roll(ids, -1)

    def grads(ck):
        m = model(kind)
        flat = torch.zeros(m.flat_numel)
        m.attach_main_grad(flat)
        m.gradient_checkpointing = ck
        m.token_logprobs(m(ids, pos, cu, 14), tgt)[0].sum().backward()
        return m, flat

    m, a = grads(False)
    assert torch.allclose(a, grads(True)[1], atol=1e-5, rtol=1e-4)
    if m.args.qk_norm:
        assert all(m.p(f"layers.{i}.{n}").main_grad.abs().sum() > 0 for i in range(2) for n in ("q_norm", "k_norm"))
    # one weight of the first layer against a difference (fp32 forward: a wide step, a loose bound)
    o = m.offsets["layers.0.wqkv"][0] + 5
    e, vals = 2e-2, []
    for s in (1, -1):
        with torch.no_grad():
            m.flat_params[o] += s * e
            vals.append(float(m.token_logprobs(m(ids, pos, cu, 14), tgt)[0].double().sum()))
            m.flat_params[o] -= s * e
    assert abs((vals[0] - vals[1]) / (2 * e) - float(a[o])) <= 2e-2 * (1 + abs(float(a[o])))


@pytest.mark.parametrize("name", ["qwen3-yarn", "llama-llama3", "llama-linear"])
def test_scaled_positions_match_transformers(name):
    import transformers as tf

    base = dict(vocab_size=128, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, max_position_embeddings=256, rms_norm_eps=1e-6, tie_word_embeddings=False)
    scal = {"yarn": YARN, "llama3": LLAMA3, "linear": {"rope_type": "linear", "factor": 2.0}}[name.split("-")[1]]
    base["rope_parameters"] = {**scal, "rope_theta": 1e4}
    torch.manual_seed(0)
    if name.startswith("qwen3"):
        cfg = tf.Qwen3Config(head_dim=16, **base)
        hf = tf.Qwen3ForCausalLM(cfg)
    else:
        cfg = tf.LlamaConfig(**base)
        hf = tf.LlamaForCausalLM(cfg)
    hf = hf.float().eval()
    args = ModelArgs.from_hf_config(cfg.to_dict())
    assert args.rope_scaling["rope_type"] == scal["rope_type"] and args.rope_theta == 1e4
    m = CausalLM(args, dtype=torch.float32, seed=None)
    hf_io.load_hf_state_dict(m, hf.state_dict())
    n = 150  # beyond the original context
    ids = torch.randint(0, 128, (n,))
    with torch.no_grad():
        got = m.logits(m(ids, torch.arange(n, dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32), n)).float()
        want = hf(ids[None]).logits[0]
    assert torch.allclose(got, want, atol=2e-4, rtol=2e-4), (got - want).abs().max()
    again = ModelArgs.from_hf_config(args.to_hf_config())
    assert again.rope_scaling == args.rope_scaling and again.rope_theta == args.rope_theta


def test_config_of_rotary_layouts():
    cfg = ModelArgs(head_dim=16, partial_rotary_factor=0.25, rope_interleaved=True).to_hf_config()
    a = ModelArgs.from_hf_config(cfg)
    assert a.rotary_dim == 4 and a.rope_interleaved and a.rope_scaling is None and a.rotates_in_pass
    assert not ModelArgs().rotates_in_pass
    plain = ModelArgs.from_hf_config({**ModelArgs().to_hf_config(), "rope_scaling": {"rope_type": "dynamic", "factor": 2.0}})
    assert plain.rope_scaling is None
    stretched = CausalLM(ModelArgs(max_position_embeddings=64, rope_scaling=YARN, num_layers=1), seed=None)
    assert stretched.rope_table("cpu").shape == (256, 64)
