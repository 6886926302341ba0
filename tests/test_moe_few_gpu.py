"""Few-token mixture-of-experts kernels against 64-bit definitions on the device."""
import pytest
import torch
from test_moe_few_cpu import experts64, make, route64

from skyrl_b200.ops import _lib, moe_few

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def check(h, rw, wgu, wd, k, norm=True, live=None):
    w, idx = moe_few.route_few(h, rw, k, norm, live=live)
    w64, i64 = route64(h, rw, k, norm)
    if live is not None:
        off = (live == 0)[:, None]
        w64, i64 = torch.where(off, 0.0, w64), torch.where(off, -1, i64)
    assert idx.dtype == torch.int32 and torch.equal(idx.long(), i64)
    # logits rounded to fp32 after the subtraction of the largest, exponential and division: 2^-20 of a weight below 1
    assert (w.double() - w64).abs().max() <= 2.0**-20
    out = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    want, bound = experts64(h, w, idx, wgu, wd)
    tol = bound + torch.finfo(BF).eps / 2 * want.abs()
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() - tol).max())
    again = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    assert torch.equal(out, again)
    return w, idx, out


SIZES = [  # T, E, k, H, F
    (1, 8, 2, 256, 128), (1, 128, 8, 512, 96), (2, 4, 4, 64, 8), (7, 33, 3, 40, 24), (16, 64, 6, 264, 120), (17, 16, 4, 128, 64),
    (33, 8, 2, 256, 128), (64, 128, 8, 256, 64), (5, 1, 1, 8, 8), (3, 1024, 16, 64, 16), (100, 20, 5, 72, 40), (256, 16, 8, 64, 32),
    (19, 200, 1, 1024, 768), (5, 8, 2, 4104, 1032), (20, 6, 3, 2056, 40), (40, 3, 2, 6152, 24), (3, 4, 2, 2048, 2048),
    (20, 1, 1, 72, 40), (32, 2, 1, 136, 24), (33, 2, 1, 136, 24), (1, 128, 8, 2048, 768), (4, 16, 8, 264, 176),
    (34, 30, 7, 552, 136), (19, 12, 3, 1000, 72), (30, 9, 4, 104, 520), (25, 40, 2, 1016, 264), (50, 4, 2, 8, 1032), (37, 7, 5, 496, 200),
]


@pytest.mark.parametrize("T,E,k,H,F", SIZES)
def test_layer(T, E, k, H, F):
    h, rw, wgu, wd = make(T, E, k, H, F, seed=T, device="cuda", dtype=BF)
    check(h, rw, wgu, wd, k, norm=(T + E) % 2 == 0)


@pytest.mark.parametrize("T", [8, 9, 24, 32, 40, 65, 256])
def test_all_tokens_on_the_same_experts(T):
    h, rw, wgu, wd = make(1, 12, 3, 96, 56, device="cuda", dtype=BF)
    h = (h + 0.01 * torch.randn(T, 96, device="cuda", dtype=torch.float32)).to(BF)
    _, idx, _ = check(h, rw, wgu, wd, 3)
    assert idx.unique().numel() <= 6


def test_strided_rows_and_dead_rows():
    h, rw, wgu, wd = make(21, 16, 4, 128, 64, device="cuda", dtype=BF)
    wide = torch.zeros(21, 200, device="cuda", dtype=BF)
    wide[:, 24:152] = h
    odd = torch.zeros(21, 131, device="cuda", dtype=BF)
    odd[:, 1:129] = h
    live = (torch.arange(21, device="cuda") % 3 != 1).to(torch.int32)
    ref = check(h, rw, wgu, wd, 4, live=live)
    assert not ref[2][1].any() and (ref[1][1] == -1).all()
    for rows in (wide[:, 24:152], odd[:, 1:129]):
        for a, b in zip(ref, check(rows, rw, wgu, wd, 4, live=live)):
            assert torch.equal(a, b)
    none = check(h, rw, wgu, wd, 4, live=torch.zeros_like(live))
    assert not none[2].any()


def test_ties_nan_repeated_and_missing_experts():
    h, rw, wgu, wd = make(6, 40, 3, 64, 32, device="cuda", dtype=BF)
    for e in (35, 39):
        rw[e] = rw[2]
    h[0] = rw[2] * 50
    h[3, 5] = float("nan")
    h[4, 7] = float("inf")
    w, idx = moe_few.route_few(h, rw, 3)
    assert idx[0].tolist() == [2, 35, 39]
    assert torch.isnan(w[3]).all() and torch.isnan(w[4]).any()
    assert ((idx >= 0) & (idx < 40)).all() and all(len(set(r)) == 3 for r in idx.tolist())
    out = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    assert torch.isnan(out[3]).all() and torch.isfinite(out[[0, 1, 2, 5]]).all()
    idx = torch.tensor([[1, 1, 7], [3, -1, 3], [40, 99, -2], [5, 5, 5], [0, 39, 39], [8, -1, 2]], device="cuda", dtype=torch.int32)
    w = torch.rand(6, 3, device="cuda") - 0.3
    w[2], w[1, 1] = float("nan"), float("inf")  # weights of slots without an expert
    h[3:5] = 1.0
    out = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    want, bound = experts64(h, w, idx, wgu, wd)
    assert ((out.double() - want).abs() <= bound + 2.0**-8 * want.abs()).all() and not out[2].any()


@pytest.mark.parametrize("E,H", [(40, 64), (128, 2048), (1000, 520)])
def test_equal_logits_summed_in_other_orders(E, H):
    """Experts whose weights are one another's in another order: all logits are equal, or one of two values, whatever
    fp32 sums make of them."""
    g = torch.Generator().manual_seed(E)
    base = torch.randn(H, generator=g).to(BF)
    rw = torch.stack([base[torch.randperm(H, generator=g)] for _ in range(E)]).cuda()
    h = torch.tensor([1.0, -0.5, 2.0**-20], dtype=BF)[:, None].expand(3, H).contiguous().cuda()
    w, idx = moe_few.route_few(h, rw, 8)
    assert torch.equal(idx, torch.arange(8, device="cuda", dtype=torch.int32).expand(3, 8)) and (w - 0.125).abs().max() <= 2.0**-20
    rw[1::2, 0] += torch.where(base.float().sum() < 0, -2.0, 2.0).to(BF).cuda()
    for norm in (True, False):
        w, idx = moe_few.route_few(h, rw, 3, norm)
        w64, i64 = route64(h, rw, 3, norm)
        assert torch.equal(idx.long(), i64) and (w.double() - w64).abs().max() <= 2.0**-20


@pytest.mark.parametrize("E,H,k", [(40, 64, 8), (128, 2048, 3), (250, 4104, 16)])
def test_logits_apart_by_less_than_a_sum_of_fp32_holds(E, H, k):
    """Two large columns cancel; what is left orders the experts and lies below the last bit of the large ones."""
    rw = torch.zeros(E, H, dtype=BF)
    rw[:, 0], rw[:, 1] = 2.0**15, -(2.0**15)
    rw[:, 2] = torch.tensor([e * 37 % E for e in range(E)]) * 2.0**-14
    rw = rw.cuda()
    for norm in (True, False):
        h = torch.ones(9, H, device="cuda", dtype=BF)
        w, idx = moe_few.route_few(h, rw, k, norm)
        w64, i64 = route64(h, rw, k, norm)
        assert torch.equal(idx.long(), i64) and (w.double() - w64).abs().max() <= 2.0**-20


@pytest.mark.parametrize("E,H", [(40, 64), (300, 520)])
def test_infinite_logits(E, H):
    """An expert with a logit of -inf is left out without spoiling its row; one of +inf comes first, and the weights are
    those of the definition (inf - inf)."""
    h, rw, *_ = make(3, E, 3, H, 8, device="cuda", dtype=BF)
    h[:, 9] = torch.tensor([1.0, 2.0, 0.5], device="cuda")
    rw[5, 9] = float("-inf")
    for norm in (True, False):
        w, idx = moe_few.route_few(h, rw, 3, norm)
        w64, i64 = route64(h, rw, 3, norm)
        assert torch.equal(idx.long(), i64) and not (idx == 5).any()
        assert (w.double() - w64).abs().max() <= 2.0**-20
    rw[7, 9] = float("inf")
    w, idx = moe_few.route_few(h, rw, 3)
    cw, cidx = moe_few.route_few(h.cpu(), rw.cpu(), 3)
    assert (idx[:, 0] == 7).all() and torch.equal(idx.cpu(), cidx) and torch.equal(torch.isnan(w).cpu(), torch.isnan(cw))


def test_capture_replays_on_new_routing():
    h, rw, wgu, wd = make(12, 32, 4, 128, 64, device="cuda", dtype=BF)

    def step():
        w, idx = moe_few.route_few(h, rw, 4)
        return moe_few.expert_ffn_few(h, w, idx, wgu, wd), idx

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):  # two graphs over the same tensors
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (1, 2):
        h.copy_(make(12, 32, 4, 128, 64, seed=seed, device="cuda", dtype=BF)[0])
        for g, (o, i) in zip(graphs, outs):
            g.replay()
            want, wi = step()
            assert torch.equal(i, wi) and torch.equal(o, want)
    assert _lib.status_read_clear() == 0


def test_no_rows_and_refusals():
    h, rw, wgu, wd = make(4, 8, 2, 64, 32, device="cuda", dtype=BF)
    w, idx = moe_few.route_few(h[:0], rw, 2)
    assert moe_few.expert_ffn_few(h[:0], w, idx, wgu, wd).shape == (0, 64)
    w, idx = moe_few.route_few(h, rw, 2)
    for a in ((h.float(), w, idx, wgu.float(), wd.float()), (h.half(), w, idx, wgu.half(), wd.half()), (h, w, idx.cpu(), wgu, wd)):
        with pytest.raises(ValueError):
            moe_few.expert_ffn_few(*a)
    with pytest.raises(ValueError):
        moe_few.route_few(h, rw.cpu(), 2)
