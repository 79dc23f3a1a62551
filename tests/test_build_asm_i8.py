"""The integer product's kernels keep their matrix instructions out of branches
that narrow EXEC (tests/test_build_asm.py says why), and their registers."""
import os
import re
import shutil

import pytest

from test_build_asm import CSRC, HIPCC, _asm, _mfma_under_narrowed_exec


@pytest.fixture(scope="module")
def i8_asm(tmp_path_factory):
    if not os.path.exists(HIPCC) and not shutil.which("hipcc"):
        pytest.skip("no hipcc")
    return _asm(os.path.join(CSRC, "apus_i8.hip"), tmp_path_factory.mktemp("asm"))


def test_no_mfma_under_narrowed_exec_i8(i8_asm):
    kernels = re.findall(r"^(_Z\d+apus_i8_(?:block|narrow)_kernel\S*):", i8_asm, re.M)
    assert len(kernels) >= 12
    assert i8_asm.count("v_mfma_i32") > 200
    assert _mfma_under_narrowed_exec(i8_asm) == {}


def test_no_scratch_i8(i8_asm):
    sizes = re.findall(r"\.private_segment_fixed_size:\s*(\d+)", i8_asm)
    assert sizes and set(sizes) == {"0"}
