"""Rotary tables are built in pieces: the same values as at once, and little memory beside the table."""
import pytest
import torch

from skyrl_b200.ops import elementwise as ew

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}


def at_once(max_pos, R, theta, device, scaling):
    inv, gain = ew.rope_frequencies(R, theta, scaling)
    ang = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv.to(device)[None, :]
    return (torch.cat([ang.cos(), ang.sin()], dim=-1) * gain).float()


def check(device, max_pos, R, scaling):
    got = ew.build_rope_table(max_pos, R, 1e4, device, scaling=scaling)
    assert got.is_contiguous() and got.dtype == torch.float32 and got.device.type == device
    assert torch.equal(got, at_once(max_pos, R, 1e4, device, scaling))


SIZES = [(1, 2), (8191, 20), (32768, 128), (32769, 128), (65535, 128), (700000, 6)]


@pytest.mark.parametrize("max_pos,R", SIZES)
@pytest.mark.parametrize("scaling", [None, YARN])
def test_values(max_pos, R, scaling):
    check("cpu", max_pos, R, scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("max_pos,R", SIZES)
@pytest.mark.parametrize("scaling", [None, YARN])
def test_values_on_the_gpu(max_pos, R, scaling):
    check("cuda", max_pos, R, scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [None, YARN])
def test_memory_beside_the_table(scaling):
    ew.build_rope_table(16384, 128, 1e4, "cuda", scaling=scaling)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    table = ew.build_rope_table(262144, 128, 1e4, "cuda", scaling=scaling)
    beside = torch.cuda.max_memory_allocated() - before - table.numel() * 4
    # angles and cosines (or sines) of 32768 positions in 64 bits, 16 MB each, the positions and the allocator's rounding
    assert beside <= 36 << 20
