"""Tensor-parallel fused decode of models whose heads go through ``ops/rotary.py``, with two shards on one GPU.

The shards take turns on the host: each runs up to its next row-parallel projection, leaves its partial sums there and
hands over, so that no kernel waits for another; the sums then stand where the peers' stores would have put them.
"""
import dataclasses
import threading
import types

import pytest
import torch

from skyrl_b200.engine.llm_engine import EngineConfig, LLMEngine, SamplingParams
from skyrl_b200.engine.tp_model import TPEngineModel
from skyrl_b200.models.decoder import PRESETS, CausalLM
from skyrl_b200.ops import _lib

pytestmark = pytest.mark.gpu
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
KINDS = {
    "plain": {},
    "norms": dict(qk_norm=True, rope_scaling=YARN),
    "norms-part": dict(qk_norm=True, partial_rotary_factor=0.5),
    "neighbours": dict(rope_interleaved=True, partial_rotary_factor=0.25),
}


class Turns:
    """Which of ``size`` threads runs; ``meet(rank, value)`` returns every rank's value once all have come by."""

    def __init__(self, size):
        self.size, self.cv, self.turn, self.left = size, threading.Condition(), 0, [[] for _ in range(size)]
        self.taken, self.failed = [0] * size, False

    def wait(self, rank):
        with self.cv:
            if not self.cv.wait_for(lambda: self.turn == rank or self.failed, timeout=120) or self.failed:
                raise RuntimeError("the other shard is gone")

    def pass_on(self, rank):
        with self.cv:
            self.turn = (rank + 1) % self.size
            self.cv.notify_all()

    def meet(self, rank, value):
        self.left[rank].append(value)
        n = self.taken[rank]
        if any(len(v) <= n for v in self.left):
            self.pass_on(rank)
            self.wait(rank)
        self.taken[rank] += 1
        return [v[n] for v in self.left]


class Shard(TPEngineModel):
    calls = 0

    def row_parallel_partials(self, x_local, w_shard, tag, dtype, channel, replayable):
        self.calls += replayable  # a projection of the fused decode step
        y = (x_local.float() @ w_shard.float().t()).to(dtype)
        return torch.stack(self.turns.meet(self.tp.rank, y))


def run_shards(full, prompts, sp, cfg):
    turns, outs, models = Turns(2), [None, None], []
    for r in range(2):
        m = Shard(full.args, types.SimpleNamespace(size=2, rank=r, fused=True, peer=None, group=None), device="cuda")
        m.load_from_full(full)
        m.turns = turns
        models.append(m)

    def work(r):
        try:
            turns.wait(r)
            outs[r] = LLMEngine(models[r], EngineConfig(**cfg)).generate(prompts, sp)
            torch.cuda.synchronize()
            turns.pass_on(r)
        except BaseException as e:
            outs[r] = e
            with turns.cv:
                turns.failed = True
                turns.cv.notify_all()

    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for o in outs:
        if isinstance(o, BaseException):
            raise o
    assert all(m.calls for m in models)
    return outs


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_two_shards_decode_what_one_model_decodes(kind):
    full = CausalLM(dataclasses.replace(PRESETS["tiny-llama-d128"], **KINDS[kind]), device="cuda", dtype=torch.bfloat16, seed=5)
    with torch.no_grad():
        for name, p in full.named_flat_views():
            if name.endswith(("q_norm", "k_norm")):
                g = torch.Generator(device="cuda").manual_seed(len(name))
                p.copy_(1 + 0.3 * torch.randn(p.shape, generator=g, device="cuda"))
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(4, 2000, (n,), generator=g).tolist() for n in (33, 5, 90, 64)]
    sp = SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True)
    cfg = dict(block_size=16, max_num_seqs=8, max_model_len=256, enforce_eager=True, num_blocks=256)
    want = LLMEngine(full, EngineConfig(**cfg)).generate(prompts, sp)
    a, b = run_shards(full, prompts, sp, cfg)
    for x, y, o in zip(a, b, want):
        assert x.token_ids == y.token_ids and x.logprobs == y.logprobs  # the shards stay in step
        # greedy decoding may fork on a near tie: the common prefix
        k = next((i for i, (s, t) in enumerate(zip(x.token_ids, o.token_ids)) if s != t), 8)
        assert k >= 1 and (torch.tensor(x.logprobs[:k]) - torch.tensor(o.logprobs[:k])).abs().max() < 5e-2
    assert _lib.status_read_clear() == 0
