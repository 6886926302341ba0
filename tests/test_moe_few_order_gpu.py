"""Routing of few tokens: the order of experts whose logits share one dominating product."""
import pytest
import torch
from test_moe_few_cpu import route64

from skyrl_b200.ops import moe_few

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("H", [64, 2048])
@pytest.mark.parametrize("first,count", [(1, 15), (1, 31), (1, 7)])
@pytest.mark.parametrize("cut", range(19, 29))
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_one_dominating_column_and_products_below_its_last_bit(H, first, count, cut, sign):
    """Expert 5: many products of less than 2^-cut of the dominating one beside them, which a sum that aligns its addends to
    the largest drops at some cut; expert 2: one product, elsewhere, of a little less than their sum."""
    E = 24
    small = 2.0**-cut * (1 - 2.0**-8)
    rw = torch.zeros(E, H, dtype=BF)
    rw[:, 0] = 1.0
    rw[:, H - 1] = -(2.0**-10)  # the others are well behind
    rw[5, first : first + count] = sign * small
    total = torch.tensor(count * small * (1 - 2.0**-7)).to(BF)
    rw[5, H - 1] = rw[2, H - 1] = 0.0
    rw[2, 48] = sign * total
    rw = rw.cuda()
    for scale in (1.0, 2.0**40, -1.0):
        h = torch.full((3, H), scale, device="cuda", dtype=BF)
        for k in (1, 2, E):
            w, idx = moe_few.route_few(h, rw, min(k, 16))
            assert torch.equal(idx.long(), route64(h, rw, min(k, 16), True)[1]), (scale, k, idx[0].tolist())


@pytest.mark.parametrize("E,H,k", [(40, 64, 8), (128, 2048, 8), (250, 4104, 16)])
@pytest.mark.parametrize("level", range(18, 30, 2))
def test_random_products_around_the_last_bit_of_a_dominating_one(E, H, k, level):
    g = torch.Generator().manual_seed(level)
    rw = (torch.randn(E, H, generator=g) * 2.0**-level).to(BF)
    h = torch.randn(33, H, generator=g).to(BF)
    rw[:, 7] = 1.0
    h[:, 7] = torch.randn(33, generator=g).abs().to(BF) + 0.5
    rw, h = rw.cuda(), h.cuda()
    for norm in (True, False):
        w, idx = moe_few.route_few(h, rw, k, norm)
        w64, i64 = route64(h, rw, k, norm)
        assert torch.equal(idx.long(), i64)
        assert (w.double() - w64).abs().max() <= 2.0**-20
