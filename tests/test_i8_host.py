"""The integer product's host side (no GPU needed): what its launchers set up."""
import ctypes as C
import re
import subprocess

import pytest

import apus_hip
from test_gpu_i8_schedules import SHAPES


def schedule(M, O, K):
    """(rows, channels, waves that split K, steps under way, threads) of a workgroup"""
    shape = (C.c_int32 * 5)()
    apus_hip.lib().apus_hip_host_i8_schedule(M, O, K, shape)
    return tuple(shape)


def test_each_kernel_has_its_own_lds_limit():
    """dynamic LDS beyond 64 KB has to be allowed kernel by kernel; a launcher does that in the
    initialiser of a static, so each kernel needs one whose name holds it"""
    out = subprocess.run(["nm", apus_hip.LIB_PATH], capture_output=True, text=True, check=True).stdout
    kernels = re.findall(r"__device_stub__(apus_i8_(?:block|narrow)_kernelI\S+)$", out, re.M)
    statics = re.findall(r" (_ZGV\S*attr)$", out, re.M)         # the guards of statics of that name
    assert len(kernels) >= 22
    for k in kernels:
        assert sum(k in s for s in statics) == 1, k


@pytest.mark.parametrize("M,O,K", [(1, 1 << 26, 2064), (1, (1 << 26) - 3, 8192), (1, (1 << 26) - 4, 8192), (1, 1 << 26, 16),
                                   (1, (1 << 26) + 1, 16), (2, 1 << 26, 16), (9, 1 << 26, 16), (9, (1 << 26) + 1, 16),
                                   ((1 << 29) + (1 << 20), 64, 16), (1 << 30, 3, 16), (0x7FFFFF00, 1, 16), (1 << 27, 40, 128),
                                   (300000, 300000, 16), (0x7FFFFF00, 1 << 26, 16)])
def test_schedules_that_a_launch_can_hold(M, O, K):
    """a launch has fewer than 2^32 threads; what no schedule holds goes to the kernel that loops"""
    rows, cols, _, _, threads = schedule(M, O, K)
    if rows:
        assert -(-M // rows) * -(-O // cols) * threads < 1 << 32
    else:
        assert O > (1 << 26) - 4 or M == 0x7FFFFF00


def test_every_schedule_is_reached():
    """The shapes of tests/test_gpu_i8_schedules.py in each schedule: steps of K a wave fewer than,
    as many as and at least two more than are under way, the last one whole and ragged."""
    seen = {}
    for M, O, K in SHAPES:
        s = schedule(M, O, K)
        steps, (rows, cols, split, depth, _) = -(-K // 128), s
        least, most = steps // split, -(-steps // split)
        how = "fewer" if most < depth else "as many" if least == most == depth else "more" if least >= depth + 2 else None
        assert M % rows or O % cols
        seen.setdefault(s, set()).add((how, K % 128 != 0))
    both = {(how, ragged) for how in ("fewer", "as many", "more") for ragged in (False, True)}
    # 8 x 32 is taken up to K 1024, which is all that its two waves have under way; four stages
    # of 128 x 128 lose to two where there are few steps
    part = {(8, 32, 2, 4, 128): {b for b in both if b[0] != "more"}, (128, 128, 1, 4, 512): {b for b in both if b[0] == "more"}}
    tiles = [(8, 16, 4, 4, 256), (8, 32, 2, 4, 128), (16, 16, 4, 4, 256), (32, 32, 2, 4, 128), (64, 32, 4, 2, 256),
             (64, 64, 1, 4, 512), (64, 128, 1, 4, 512), (128, 128, 1, 4, 512), (128, 128, 1, 2, 512), (256, 128, 1, 3, 512),
             (256, 256, 1, 2, 512)]
    assert set(seen) == set(tiles)
    for s in tiles:
        assert part.get(s, both) <= seen[s], (s, part.get(s, both) - seen[s])


def test_schedules_of_one_row():
    """the widths of the one-row schedule, which tests/test_gpu_i8.py runs at K 16 to 8192"""
    assert [schedule(1, 130, K)[:2] for K in (16, 1024, 1040, 2048, 2064, 8192)] == [(1, 16), (1, 16), (1, 8), (1, 8), (1, 4), (1, 4)]
