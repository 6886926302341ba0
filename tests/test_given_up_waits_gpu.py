"""Kernels that start while the status word is set give up their waits early: the call ends, the status stays for the host
to read, copies under way land in their own buffers, and what runs beside and after it is right.

The status is set as in the test of a barrier that runs out: one that the absent second rank never signals.
"""
import ctypes

import pytest
import torch
from test_moe_few_cpu import make

from skyrl_b200.ops import _lib, elementwise, moe_few, rotary

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


@pytest.mark.parametrize("D,R,dtype", [(128, 128, BF), (80, 20, torch.float16), (64, 64, torch.float32)])
def test_row_pipeline(status, D, R, dtype):
    T, nq, nkv = 8192, 8, 2
    g = torch.Generator(device="cuda").manual_seed(D)
    x, dy = (torch.randn(T, (nq + 2 * nkv) * D, generator=g, device="cuda").to(dtype) for _ in range(2))
    qw, kw = (torch.rand(D, generator=g, device="cuda").to(dtype) + 0.5 for _ in range(2))
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    table = elementwise.build_rope_table(T, R, 1e4, "cuda")

    def step():
        a = [t.clone().requires_grad_() for t in (x, qw, kw)]
        y = rotary.qk_norm_rope(*a, pos, table, nq, nkv, D, 1e-6)
        return [y.detach(), *torch.autograd.grad(y, a, dy)]

    want = step()
    status()
    for _ in range(10):
        step()
        beside = rotary.rotary(x[:64], pos[:64], table, nq + nkv, D)  # too few rows for the pipeline
    torch.cuda.synchronize()
    assert _lib.status_read_clear() == 0x901
    assert torch.equal(beside, rotary.rotary(x, pos, table, nq + nkv, D)[:64])
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    assert _lib.status_read_clear() == 0
