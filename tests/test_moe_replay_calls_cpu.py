"""The expert layer hands its routing out only while something records or replays it."""
import pytest
import torch

from skyrl_b200.models import moe, router_replay


@pytest.fixture
def calls(monkeypatch):
    seen, real = [], router_replay.on_route

    def spy(layer, idx):
        seen.append((layer, idx.dtype))
        return real(layer, idx)

    monkeypatch.setattr(router_replay, "on_route", spy)
    return seen


def test_routing_is_handed_out_only_when_asked_for(calls):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    h, rw, wgu, wd = r(5, 16), r(6, 16), r(6, 16, 16), r(6, 16, 8)
    out = moe.moe_ffn(h, rw, wgu, wd, 2, layer=3)
    assert not calls
    with router_replay.record_routing() as store:
        moe.moe_ffn(h, rw, wgu, wd, 2, layer=3)
    assert calls == [(3, torch.int64)] and store[3].shape == (5, 2) and store[3].dtype == torch.int64
    table = torch.full((5, 4, 2), router_replay.PAD)
    table[:, 3] = store[3]
    with router_replay.replay_routing(table):
        assert torch.allclose(moe.moe_ffn(h, rw, wgu, wd, 2, layer=3), out, atol=1e-6)
    assert len(calls) == 2
    router_replay.set_replay(table)
    try:
        moe.moe_ffn(h, rw, wgu, wd, 2, layer=3)
    finally:
        router_replay.set_replay(None)
    assert len(calls) == 3
    moe.moe_ffn(h, rw, wgu, wd, 2, layer=3)
    assert len(calls) == 3
