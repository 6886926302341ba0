"""Mixture-of-experts layer for a few tokens: the CPU formulation against 64-bit definitions; refusals."""
import pytest
import torch

from skyrl_b200.ops import moe_few


def route64(h, rw, k, norm):
    """(weights, ids) from the definition, ties to the lower expert."""
    z = h.double() @ rw.double().t()
    p = torch.softmax(z, -1)
    ids = []
    left = z.clone()
    for _ in range(k):
        top = left.max(-1, keepdim=True).values
        e = torch.where(left == top, torch.arange(z.shape[1], device=z.device), z.shape[1]).min(-1).values
        ids.append(e)
        left.scatter_(1, e[:, None], float("-inf"))
    ids = torch.stack(ids, 1)
    w = p.gather(1, ids)
    return (w / w.sum(-1, keepdim=True) if norm else w), ids


def experts64(h, w, idx, wgu, wd):
    """(out, bound): fp64 outputs and, for each, a bound on what rounding the activations to the rows' type and fp32 sums
    can do to it."""
    T, k = idx.shape
    F, H = wd.shape[2], h.shape[1]
    u = torch.finfo(h.dtype).eps / 2
    out, bound = (torch.zeros(T, H, dtype=torch.float64, device=h.device) for _ in range(2))
    for t in range(T):
        for s in range(k):
            e = int(idx[t, s])
            if not 0 <= e < wd.shape[0]:
                continue
            g, x = wgu[e].double(), h[t].double()
            gu, mag = g @ x, g.abs() @ x.abs()
            sig = torch.sigmoid(gu[:F])
            act = gu[:F] * sig * gu[F:]
            # sums of H products in fp32, whatever their order (one unit of 2^-23 a step covers truncating adders);
            # |silu'| < 1.1, and 2^-18 for the exponential and the products around it
            d = H * 2.0**-23 * mag
            err = u * act.abs() + 2.0**-18 * act.abs() + 1.1 * d[:F] * (gu[F:].abs() + d[F:]) + (gu[:F] * sig).abs() * d[F:]
            y, ymag = wd[e].double() @ act, wd[e].double().abs()
            out[t] += float(w[t, s]) * y
            bound[t] += abs(float(w[t, s])) * (ymag @ err + (F * 2.0**-23 + k * 2.0**-23) * (ymag @ act.abs()))
    return out, bound


def make(T, E, k, H, F, seed=0, device="cpu", dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    h, rw = r(T, H).to(dtype), (r(E, H) * 1.5 / H**0.5).to(dtype)
    return [t.to(device) for t in (h, rw, (r(E, 2 * F, H) / H**0.5).to(dtype), (r(E, H, F) / F**0.5).to(dtype))]


@pytest.mark.parametrize("T,E,k,H,F", [(1, 8, 2, 32, 16), (5, 6, 6, 24, 10), (9, 33, 3, 16, 8), (3, 1, 1, 8, 8)])
@pytest.mark.parametrize("norm", [True, False])
def test_layer_matches_64_bits(T, E, k, H, F, norm):
    h, rw, wgu, wd = make(T, E, k, H, F)
    w, idx = moe_few.route_few(h, rw, k, norm)
    w64, i64 = route64(h, rw, k, norm)
    assert torch.equal(idx.long(), i64) and (w.double() - w64).abs().max() <= 2.0**-20
    out = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    want, bound = experts64(h, w, idx, wgu, wd)
    assert ((out.double() - want).abs() <= bound + 2.0**-24 * want.abs()).all()


def test_ties_dead_rows_and_nan():
    h, rw, wgu, wd = make(4, 8, 3, 16, 8)
    rw[5] = rw[2]
    rw[7] = rw[2]
    h[0] = rw[2] * 50  # experts 2, 5 and 7 tie at the top
    h[3, 0] = float("nan")
    live = torch.tensor([1, 0, 1, 1], dtype=torch.int32)
    w, idx = moe_few.route_few(h, rw, 3, True, live=live)
    assert idx[0].tolist() == [2, 5, 7] and torch.allclose(w[0], torch.full((3,), 1 / 3))
    assert idx[1].tolist() == [-1] * 3 and w[1].tolist() == [0.0] * 3
    assert torch.isnan(w[3]).all() and ((idx[3] >= 0) & (idx[3] < 8)).all() and len(set(idx[3].tolist())) == 3
    out = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    assert float(out[1].abs().sum()) == 0 and torch.isnan(out[3]).all() and torch.isfinite(out[[0, 2]]).all()


def test_repeated_and_missing_experts():
    h, rw, wgu, wd = make(3, 4, 2, 16, 8)
    idx = torch.tensor([[1, 1], [3, -1], [9, 4]], dtype=torch.int32)
    w = torch.tensor([[0.25, 0.5], [2.0, 1.0], [1.0, 1.0]])
    out = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    one = moe_few.expert_ffn_few(h, torch.ones(3, 1), torch.tensor([[1], [3], [0]], dtype=torch.int32), wgu, wd)
    assert torch.allclose(out[0], 0.75 * one[0], atol=1e-6) and torch.allclose(out[1], 2 * one[1], atol=1e-6)
    assert float(out[2].abs().sum()) == 0


def test_refusals():
    h, rw, wgu, wd = make(4, 8, 2, 16, 8)
    w, idx = moe_few.route_few(h, rw, 2)
    for a in ((h, rw, 0), (h, rw, 9), (h, rw, 17), (h, rw[:, :8], 2), (h.half(), rw, 2), (h, rw.t().contiguous().t(), 2), (h[0], rw, 2),
              (h.clone().requires_grad_(), rw, 2), (h, torch.zeros(1025, 16), 2)):
        with pytest.raises(ValueError):
            moe_few.route_few(*a)
    for live in (torch.ones(4), torch.ones(3, dtype=torch.int32), torch.ones(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            moe_few.route_few(h, rw, 2, live=live)
    for a in ((h, w, idx.long(), wgu, wd), (h, w.double(), idx, wgu, wd), (h, w[:2], idx, wgu, wd), (h, w, idx, wgu[:, :8], wd),
              (h, w, idx, wgu, wd[:4]), (h, w, idx, wgu.half(), wd), (h, w, idx, wgu, wd.transpose(1, 2).contiguous().transpose(1, 2)),
              (h, w, idx, wgu, wd.clone().requires_grad_())):
        with pytest.raises(ValueError):
            moe_few.expert_ffn_few(*a)
    big = torch.zeros(300, 16), torch.zeros(300, 8), torch.zeros(300, 8, dtype=torch.int32)
    with pytest.raises(ValueError):
        moe_few.expert_ffn_few(*big, wgu, wd)


def test_supports():
    assert moe_few.supports(64, 128, 8, 2048, 768) and moe_few.supports(256, 128, 8, 2048, 768)
    for bad in ((257, 128, 8, 2048, 768), (4, 2000, 8, 64, 64), (4, 64, 17, 64, 64), (4, 4, 5, 64, 64), (4, 8, 2, 60, 64), (4, 8, 2, 64, 60)):
        assert not moe_few.supports(*bad)


def test_routing_weights_with_gradients_are_refused():
    h, rw, wgu, wd = make(3, 4, 2, 16, 8)
    w, idx = moe_few.route_few(h, rw, 2)
    with pytest.raises(ValueError, match="gradient"):
        moe_few.expert_ffn_few(h, w.clone().requires_grad_(), idx, wgu, wd)
    with torch.no_grad():
        moe_few.expert_ffn_few(h, w.clone().requires_grad_(), idx, wgu, wd)
