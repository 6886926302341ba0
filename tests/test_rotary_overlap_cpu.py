"""Rows on their way into the cache: which ``out`` may share memory with them."""
import pytest
import torch

from skyrl_b200.ops import elementwise as ew
from skyrl_b200.ops import rotary

D, NQ, NKV = 8, 2, 1
W = (NQ + 2 * NKV) * D


def call(x, out):
    T = x.shape[0]
    kc, vc = torch.zeros(4, 4, NKV, D), torch.zeros(4, 4, NKV, D)
    return rotary.qk_rope_cache(x, torch.arange(T, dtype=torch.int32), ew.build_rope_table(16, D, 1e4, "cpu"), kc, vc,
                                torch.arange(T, dtype=torch.int32), NQ, NKV, D, out=out)


@pytest.mark.parametrize("T", [1, 2, 3])
def test_columns_apart_and_an_out_that_starts_with_them(T):
    """``x`` takes every other column of a buffer and ``out`` its first ones: not the same elements, for one row too."""
    buf = torch.randn(T, 2 * W)
    with pytest.raises(ValueError, match="other elements"):
        call(buf[:, ::2], buf[:, :W])
    want = call(buf[:, ::2].clone(), None)
    assert torch.equal(call(buf[:, ::2], torch.empty(T, W)), want)


@pytest.mark.parametrize("T", [1, 2, 3])
def test_the_same_rows(T):
    buf = torch.randn(T, 2 * W)
    x = buf[:, :W]
    want = call(x.clone(), None)
    assert torch.equal(call(x, x), want) and torch.equal(buf[:, :W], want)
