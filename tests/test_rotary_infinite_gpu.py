"""Infinities in the part of a head that is not rotated stay with their element, for few rows and for many."""
import pytest
import torch

from skyrl_b200.ops import elementwise as ew
from skyrl_b200.ops import rotary

pytestmark = pytest.mark.gpu
NQ, NKV = 4, 2


@pytest.mark.parametrize("D,R", [(128, 64), (80, 20), (96, 24), (64, 4)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [3, 20000])
def test_unrotated_infinities(D, R, inter, dtype, T):
    g = torch.Generator(device="cuda").manual_seed(D)
    W = (NQ + 2 * NKV) * D
    x, dy = (torch.randn(T, W, generator=g, device="cuda").to(dtype) for _ in range(2))
    qw, kw = (torch.rand(D, generator=g, device="cuda").to(dtype) + 0.5 for _ in range(2))
    pos = torch.arange(T, device="cuda", dtype=torch.int32) % 512
    table = ew.build_rope_table(512, R, 1e4, "cuda")
    at = [(0, 0, D - 1), (T - 1, NQ, R), (T // 2, 1, (R + D) // 2)]  # row, head, element
    bad = x.clone()
    for t, h, e in at:
        bad[t, h * D + e] = float("inf")

    y = rotary.rotary(x, pos, table, NQ + NKV, D, interleaved=inter)
    z = rotary.rotary(bad, pos, table, NQ + NKV, D, interleaved=inter)
    assert torch.equal(y.isfinite().logical_not(), torch.zeros_like(y, dtype=torch.bool))
    assert torch.equal(z != y, bad != x) and torch.equal(z.isinf(), bad.isinf())

    # the head's root mean square is infinite: its finite elements become zero, the infinite one inf / inf
    y = rotary.qk_norm_rope(x, qw, kw, pos, table, NQ, NKV, D, 1e-6, interleaved=inter)
    z = rotary.qk_norm_rope(bad, qw, kw, pos, table, NQ, NKV, D, 1e-6, interleaved=inter)
    for t, h, e in at:
        head = z[t, h * D : (h + 1) * D]
        nan = torch.zeros(D, dtype=torch.bool, device="cuda")
        nan[e] = True
        assert torch.equal(head.isnan(), nan) and not head[~nan].any()
        z[t, h * D : (h + 1) * D] = y[t, h * D : (h + 1) * D]
    assert torch.equal(z, y)

    # an infinite gradient reaches its own element of the weight's gradient and all of its head's
    leaves = [v.clone().requires_grad_() for v in (x, qw, kw)]
    out = rotary.qk_norm_rope(*leaves, pos, table, NQ, NKV, D, 1e-6, interleaved=inter)
    bad = dy.clone()
    for t, h, e in at:
        bad[t, h * D + e] = float("inf")
    want = torch.autograd.grad(out, leaves, dy, retain_graph=True)
    got = torch.autograd.grad(out, leaves, bad)
    for part, heads in ((1, range(NQ)), (2, range(NQ, NQ + NKV))):
        hit = torch.zeros(D, dtype=torch.bool, device="cuda")
        for t, h, e in at:
            if h in heads:
                hit[e] = True
        assert not got[part][hit].isfinite().any() and torch.equal(got[part][~hit], want[part][~hit])
    for t, h, e in at:
        assert not got[0][t, h * D : (h + 1) * D].isfinite().any()
        got[0][t, h * D : (h + 1) * D] = want[0][t, h * D : (h + 1) * D]
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("D,R,dtype", [(128, 64, torch.bfloat16), (80, 20, torch.float16)])
def test_unrotated_infinities_on_their_way_into_the_cache(D, R, dtype):
    """Rows in place, and their cache rows, many at once: what a few rows at a time give."""
    T = 20000
    g = torch.Generator(device="cuda").manual_seed(R)
    x = torch.randn(T, (NQ + 2 * NKV) * D, generator=g, device="cuda").to(dtype)
    qw, kw = (torch.rand(D, generator=g, device="cuda").to(dtype) + 0.5 for _ in range(2))
    rows = torch.randint(0, T, (40,), generator=g, device="cuda")
    x[rows, torch.randint(0, NQ + NKV, (40,), generator=g, device="cuda") * D + D - 1 - torch.arange(40, device="cuda") % (D - R)] = float("-inf")
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    table = ew.build_rope_table(T, R, 1e4, "cuda")

    def caches():
        return [torch.zeros(T // 32, 32, NKV, D, device="cuda", dtype=dtype) for _ in range(2)]

    kc, vc = caches()
    got = x.clone()
    rotary.qk_rope_cache(got, pos, table, kc, vc, pos, NQ, NKV, D, q_norm=qw, k_norm=kw, out=got)
    kc2, vc2 = caches()
    at = rows.unique()
    want = rotary.qk_rope_cache(x[at], pos[at], table, kc2, vc2, pos[at].contiguous(), NQ, NKV, D, q_norm=qw, k_norm=kw)
    eq = lambda a, b: bool(((a == b) | (a.isnan() & b.isnan())).all())  # noqa: E731
    tol = 2 * torch.finfo(dtype).eps  # the two forms multiply in another order: a rounding apart, of a value at most 2 |n|
    assert torch.equal(got[at].isnan(), want.isnan()) and got[at].isnan().sum() == len(rows)
    scale = want.nan_to_num().abs().amax(-1, keepdim=True)
    assert ((got[at].nan_to_num() - want.nan_to_num()).abs() <= tol * scale).all()
    part = [slice(0, NQ * D), slice(NQ * D, (NQ + NKV) * D), slice((NQ + NKV) * D, None)]
    assert eq(kc.view(T, -1), got[:, part[1]]) and eq(vc.view(T, -1), x[:, part[2]]) and eq(got[:, part[2]], x[:, part[2]])
