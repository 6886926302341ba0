"""Rotary variants, head norms, cache rows, paged layout and few-token experts together in models and engine on the GPU."""
import contextlib
import dataclasses
import types

import pytest
import torch

from skyrl_b200.engine.llm_engine import EngineConfig, LLMEngine, SamplingParams
from skyrl_b200.models import moe, router_replay
from skyrl_b200.models.decoder import PRESETS, CausalLM
from skyrl_b200.ops import _lib

pytestmark = pytest.mark.gpu
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
KINDS = {
    "dense-norms": dataclasses.replace(PRESETS["tiny-llama-d128"], qk_norm=True, rope_scaling=YARN),
    "dense-part": dataclasses.replace(PRESETS["tiny-llama-d128"], rope_interleaved=True, partial_rotary_factor=0.5),
    "experts": dataclasses.replace(PRESETS["tiny-moe"], rope_scaling=YARN, num_heads=4, num_kv_heads=2),
}


def model(kind, seed=5):
    m = CausalLM(KINDS[kind], device="cuda", dtype=torch.bfloat16, seed=seed)
    with torch.no_grad():
        for name, p in m.named_flat_views():
            if name.endswith(("q_norm", "k_norm")):
                g = torch.Generator(device="cuda").manual_seed(len(name))
                p.copy_(1 + 0.3 * torch.randn(p.shape, generator=g, device="cuda"))
    return m


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_engine_graphs_eager_and_full_forward_agree(kind):
    m = model(kind)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(4, 1000, (n,), generator=g).tolist() for n in (40, 7, 130, 64, 1)]
    sp = SamplingParams(max_tokens=20, temperature=0.0, ignore_eos=True)
    outs = {}
    for eager in (True, False):
        eng = LLMEngine(m, EngineConfig(block_size=16, max_num_seqs=8, max_model_len=256, sync_interval=4, enforce_eager=eager,
                                        num_blocks=256))
        outs[eager] = eng.generate(prompts, sp)
        if not eager:
            assert eng.stats["graph_replays"] > 0
    for a, b in zip(outs[True], outs[False]):
        assert a.token_ids == b.token_ids
        assert torch.allclose(torch.tensor(a.logprobs), torch.tensor(b.logprobs), atol=1e-3)
    for p, o in zip(prompts, outs[False]):
        toks = p + o.token_ids
        ids = torch.tensor(toks, device="cuda", dtype=torch.int32)
        with torch.no_grad():
            h = m(ids, torch.arange(len(toks), device="cuda", dtype=torch.int32),
                  torch.tensor([0, len(toks)], device="cuda", dtype=torch.int32), len(toks))
            lp, _ = m.token_logprobs(h[len(p) - 1 : -1], ids[len(p):])
        assert (lp.cpu() - torch.tensor(o.logprobs)).abs().max() < 5e-2
    assert _lib.status_read_clear() == 0


def test_fused_decode_of_a_model_with_head_norms():
    m = model("dense-norms")
    prompts = [list(range(4, 4 + n)) for n in (33, 5, 90, 64)]
    sp = SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True)
    outs = [LLMEngine(m, EngineConfig(block_size=16, max_num_seqs=8, max_model_len=256, enforce_eager=True, num_blocks=256,
                                      fused_decode=f)).generate(prompts, sp) for f in (False, True)]
    for a, b in zip(*outs):  # greedy decoding may fork on a near-tie: the common prefix
        k = next((i for i, (x, y) in enumerate(zip(a.token_ids, b.token_ids)) if x != y), 8)
        assert k >= 1 and (torch.tensor(a.logprobs[:k]) - torch.tensor(b.logprobs[:k])).abs().max() < 5e-2


def test_prefix_cache_reads_what_the_launch_wrote():
    m = model("dense-norms")
    shared = list(range(10, 75))
    prompts = [shared + [200 + i, 300 + i] for i in range(4)]
    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    cfg = dict(block_size=16, max_num_seqs=4, max_model_len=128, num_blocks=64, enforce_eager=True)
    want = LLMEngine(m, EngineConfig(**cfg)).generate(prompts, sp)
    eng = LLMEngine(m, EngineConfig(**cfg, enable_prefix_caching=True))
    got = eng.generate(prompts[:1], sp) + eng.generate(prompts[1:], sp)
    assert eng.stats["prefix_cached_tokens"] > 0
    for a, b in zip(want, got):
        assert (torch.tensor(a.logprobs[:1]) - torch.tensor(b.logprobs[:1])).abs().max() < 5e-2


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_training_gradients_match_fp32_on_the_cpu(kind):
    m = model(kind)
    ref = CausalLM(m.args, device="cpu", dtype=torch.float32, seed=None)
    ref.flat_params.copy_(m.flat_params.float().cpu())
    lens = [200, 37, 129]
    g = torch.Generator().manual_seed(2)
    ids, tgt = (torch.randint(0, m.args.vocab_size, (sum(lens),), generator=g) for _ in range(2))
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32)
    cu = torch.tensor([0, 200, 237, 366], dtype=torch.int32)
    # a token next to a border may take another expert in bf16: both models run through the fp32 model's experts
    with router_replay.record_routing() as store, torch.no_grad():
        ref(ids, pos, cu, max(lens))
    table = router_replay.stack_recorded(store) if kind == "experts" else None
    for mod, dev in ((ref, "cpu"), (m, "cuda")):
        with router_replay.replay_routing(table.to(dev)) if table is not None else contextlib.nullcontext():
            lp, _ = mod.token_logprobs(mod(ids.to(dev), pos.to(dev), cu.to(dev), max(lens)), tgt.to(dev))
            lp.sum().backward()
    for n, p in m.named_flat_views():
        gr = ref.p(n).grad
        if gr.abs().max() > 0:
            assert rel(p.grad.cpu(), gr) < 8e-2, n
    assert _lib.status_read_clear() == 0


def test_expert_layer_paths_agree_and_dead_rows_are_zero():
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    T, E, k, H, F = 50, 16, 4, 256, 128
    h, rw, wgu, wd = rnd(T, H), rnd(E, H) * 0.1, rnd(E, 2 * F, H) * 0.06, rnd(E, H, F) * 0.09
    live = (torch.arange(T, device="cuda") % 5 > 0).to(torch.int32)
    with torch.no_grad():
        assert moe._takes_few(h, rw, wgu, wd, k)
        few = moe.moe_ffn(h, rw, wgu, wd, k)
        dead = moe.moe_ffn(h, rw, wgu, wd, k, live=live)
        old, moe.FEW_ROWS = moe.FEW_ROWS, 0
        try:
            many = moe.moe_ffn(h, rw, wgu, wd, k)
        finally:
            moe.FEW_ROWS = old
        with router_replay.record_routing() as store:
            recorded = moe.moe_ffn(h, rw, wgu, wd, k, layer=0)
        table = router_replay.stack_recorded(store)
        with router_replay.replay_routing(table):
            replayed = moe.moe_ffn(h, rw, wgu, wd, k, layer=0)
    # the grouped path also rounds gate, up and the experts' outputs: a few bf16 half steps of the result's size
    assert rel(few, many) < 4 * 2.0**-8
    on = live.bool()
    assert torch.equal(dead[on], few[on]) and not dead[~on].any()
    assert torch.equal(recorded, few) and rel(replayed, few) < 2.0**-8
    # rows that need gradients train
    hg = h.clone().requires_grad_()
    moe.moe_ffn(hg, rw, wgu, wd, k).float().sum().backward()
    assert hg.grad is not None and torch.isfinite(hg.grad).all()


def test_replayed_routing_with_gaps_and_dead_rows():
    """Rows without a replayed choice keep their own; a dead row has none and comes out zero."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    T, E, k, H, F = 6, 8, 2, 64, 32
    h, rw, wgu, wd = r(T, H), r(E, H), r(E, 2 * F, H) / 8, r(E, H, F) / 8
    live = torch.tensor([1, 0, 1, 0, 1, 1], device="cuda", dtype=torch.int32)
    routes = torch.randint(0, E, (T, 1, k), generator=g, device="cuda", dtype=torch.int16)
    routes[1], routes[2] = router_replay.PAD, router_replay.PAD
    with torch.no_grad(), router_replay.replay_routing(routes):
        out = moe.moe_ffn(h, rw, wgu, wd, k, layer=0, live=live)
    with torch.no_grad():
        own = moe.moe_ffn(h, rw, wgu, wd, k, layer=0)
        forced = moe.moe_ffn(h, rw, wgu, wd, k, routed_indices=routes[:, 0].clamp_min(0))
    assert not out[1].any() and torch.equal(out[[0, 3, 4, 5]], forced[[0, 3, 4, 5]])
    # the row's own weights are taken from the replay's softmax (2^-20 of a weight apart, then one bf16 rounding)
    assert ((out[2] - own[2]).abs() <= 2.0**-7 * own[2].abs().max()).all() and torch.isfinite(out).all()


def test_fake_int4_experts_are_not_taken_by_the_path_for_few_tokens():
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    h, rw, wgu, wd = r(6, 128), r(8, 128), r(8, 128, 128) / 11, r(8, 128, 64) / 8
    qat = types.SimpleNamespace(enabled=True, group_size=32, scale_divisor=7.0, q_min=-7.0)
    frozen = moe.moe_ffn(h, rw, wgu, wd, 2, qat=qat)  # gradients are on, nothing needs one
    trained = moe.moe_ffn(h, rw, wgu.requires_grad_(), wd.requires_grad_(), 2, qat=qat)
    assert torch.equal(frozen, trained)
    with torch.no_grad():
        assert not torch.equal(frozen, moe.moe_ffn(h, rw, wgu, wd, 2, qat=qat))
