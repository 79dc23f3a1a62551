"""The integer product's host side (no GPU needed): what its launchers set up."""
import ctypes as C
import re
import subprocess

import pytest

import apus_hip


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
