"""The weight ring of the few-token expert kernel: sizes from the library's own host code, walked as its consumers do."""
import ctypes

import pytest

from skyrl_b200.ops import _lib

SHARED = 227 * 1024  # bytes a CTA may have
CONSUMERS, STEPS = 8, 12  # warps that consume, and the most 32-column steps of a warp's share where groups are smaller than that


def ring(n, E, H):
    out = [ctypes.c_int() for _ in range(5)]
    code = _lib.kernels().sb_moe_few_ring(n, E, H, *map(ctypes.byref, out))
    return code, [v.value for v in out]


@pytest.mark.parametrize("n,E", [(1, 1), (8, 128), (512, 128), (238, 104), (2048, 1024), (2048, 1), (1, 1024)])
def test_a_stage_returns_to_the_group_that_used_it_last(n, E):
    """Copies land in any order: a group may wait for a stage's phase only when it has itself seen the phase before."""
    seen = set()
    for H in [*range(8, 4200, 8), 8192, 16392, 204808]:
        code, (stages, pieces, piece, groups, smem) = ring(n, E, H)
        assert code == 0 and groups in (1, 2, 4, 8) and smem + 2 * 8 * stages <= SHARED
        assert smem >= stages * 16 * piece and pieces * piece >= H > (pieces - 1) * piece and (16 * piece) % 16 == 0
        assert (piece + 31) // 32 <= CONSUMERS // groups * (STEPS if groups > 1 else 8)
        assert groups == 1 or pieces == 1
        seen.add(groups)
        if groups == 1:  # the group meets every stage in turn
            assert stages >= 2
            continue
        last = {}  # stage -> group that used it last
        for item in range(3 * stages * groups):
            for half in range(2):
                stage = (2 * item + half) % stages
                assert last.setdefault(stage, item % groups) == item % groups, (H, stages, groups)
        # a group starts on the stages of its first item without a turn around the ring
        assert 2 * groups <= stages
    assert seen == {1, 2, 4, 8}


def test_ring_refusals():
    assert all(ring(*a)[0] == 1 for a in ((0, 4, 64), (2049, 4, 64), (4, 0, 64), (4, 1025, 64), (4, 4, 0), (4, 4, 60)))
