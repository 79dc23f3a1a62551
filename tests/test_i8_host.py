"""The integer product's host side (no GPU needed): what its launchers set up."""
import re
import subprocess

import apus_hip


def test_each_kernel_has_its_own_lds_limit():
    """dynamic LDS beyond 64 KB has to be allowed kernel by kernel; a launcher does that in the
    initialiser of a static, so each kernel needs one whose name holds it"""
    out = subprocess.run(["nm", apus_hip.LIB_PATH], capture_output=True, text=True, check=True).stdout
    kernels = re.findall(r"__device_stub__(apus_i8_(?:block|narrow)_kernelI\S+)$", out, re.M)
    statics = re.findall(r" (_ZGV\S*attr)$", out, re.M)         # the guards of statics of that name
    assert len(kernels) >= 22
    for k in kernels:
        assert sum(k in s for s in statics) == 1, k
