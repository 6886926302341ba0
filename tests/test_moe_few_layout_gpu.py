"""Few-token experts: rows and weights at strides and addresses that a 16-byte read does not allow."""
import pytest
import torch
from test_moe_few_cpu import make

from skyrl_b200.models import moe
from skyrl_b200.ops import moe_few

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def at_offset(t, by):
    """The same values, contiguous, ``by`` elements behind a 16-byte boundary."""
    buf = torch.zeros(t.numel() + 16, device=t.device, dtype=t.dtype)
    out = buf[by : by + t.numel()].view(t.shape)
    assert out.data_ptr() % 16 == 2 * by % 16
    return out.copy_(t)


@pytest.mark.parametrize("T", [1, 2, 5])
@pytest.mark.parametrize("place", ["odd stride", "odd start", "columns apart", "one row for all"])
def test_rows(T, place):
    h, rw, wgu, wd = make(T, 16, 4, 64, 32, device="cuda", dtype=BF)
    if place == "odd stride":
        buf = torch.zeros(T, 68 + 1, device="cuda", dtype=BF)
        rows = buf[:, :64]
        rows.copy_(h)
    elif place == "odd start":
        rows = at_offset(h, 3)
    elif place == "columns apart":
        rows = torch.zeros(T, 128, device="cuda", dtype=BF)[:, ::2]
        rows.copy_(h)
    else:
        h = h[:1].expand(T, 64).contiguous()
        rows = h[:1].expand(T, 64)
    w, idx = moe_few.route_few(h, rw, 4)
    for a, b in zip((w, idx), moe_few.route_few(rows, rw, 4)):
        assert torch.equal(a, b)
    assert torch.equal(moe_few.expert_ffn_few(h, w, idx, wgu, wd), moe_few.expert_ffn_few(rows, w, idx, wgu, wd))


def test_weights():
    h, rw, wgu, wd = make(6, 16, 4, 64, 32, device="cuda", dtype=BF)
    w, idx = moe_few.route_few(h, rw, 4)
    with pytest.raises(ValueError, match="boundary"):
        moe_few.route_few(h, at_offset(rw, 1), 4)
    for ws in ((at_offset(wgu, 4), wd), (wgu, at_offset(wd, 7))):
        with pytest.raises(ValueError, match="boundary"):
            moe_few.expert_ffn_few(h, w, idx, *ws)
    # the layer routes such a model through the grouped GEMMs where it can
    with torch.no_grad():
        assert moe._takes_few(h, rw, wgu, wd, 4) and not moe._takes_few(h, at_offset(rw, 1), wgu, wd, 4)
        a, b = moe.moe_ffn(h, rw, wgu, wd, 4, few_tokens=False), moe.moe_ffn(h, at_offset(rw, 1), wgu, wd, 4)
    assert torch.equal(a, b)
