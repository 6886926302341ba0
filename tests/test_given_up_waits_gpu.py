"""Kernels that start while the status word is set give up their waits early: the call ends, the status stays for the host
to read, copies under way land in their own buffers, and what runs beside and after it is right.

The status is set as in the test of a barrier that runs out: one that the absent second rank never signals.
"""
import ctypes

import pytest
import torch
from test_moe_few_cpu import make

from skyrl_b200.ops import _lib, moe_few

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture
def status():
    """Sets the status word on the current stream."""
    from skyrl_b200.parallel import peer

    lib = peer._k()
    assert _lib.status_read_clear() == 0
    pads = [torch.zeros(64, device="cuda", dtype=torch.int32) for _ in range(2)]

    def set_():
        ptrs = (ctypes.c_void_p * 2)(*(p.data_ptr() for p in pads))
        _lib.check(lib.sb_peer_barrier(ptrs, 0, 2, 0, 1, int(0.05e9), _lib.stream_ptr()), "sb_peer_barrier")

    yield set_
    torch.cuda.synchronize()
    _lib.status_read_clear()


# one, two, four and eight consumer groups; rows of two pieces; few entries of narrow and of wide experts
@pytest.mark.parametrize("T,E,k,H,F", [(64, 32, 8, 2048, 256), (64, 64, 8, 1288, 264), (64, 64, 8, 768, 384), (64, 128, 8, 256, 256),
                                       (20, 6, 3, 4104, 264), (1, 128, 8, 2048, 768), (2, 16, 8, 264, 176)])
def test_experts(status, T, E, k, H, F):
    h, rw, wgu, wd = make(T, E, k, H, F, device="cuda", dtype=BF)
    w, idx = moe_few.route_few(h, rw, k)
    want = moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    status()
    for _ in range(20):
        moe_few.expert_ffn_few(h, w, idx, wgu, wd)
    beside = moe_few.route_few(h, rw, k)
    torch.cuda.synchronize()
    assert torch.equal(beside[0], w) and torch.equal(beside[1], idx)
    assert _lib.status_read_clear() == 0x901  # the barrier's code: the first wait that gave up
    assert torch.equal(moe_few.expert_ffn_few(h, w, idx, wgu, wd), want)
    assert _lib.status_read_clear() == 0
