"""Integer products whose tiles pass what a launch holds in the schedule that would be the fastest."""
import numpy as np
import pytest

import rowops as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,O,K", [(1 << 30, 3, 16), ((1 << 29) + (1 << 20) + 5, 33, 16)])
def test_i8_more_rows_than_the_smallest_tiles_hold(hip, rng, M, O, K):
    L = hip.lib()
    n = 70
    da, ds, do = hip.DevBuf(M * K), hip.DevBuf(M * 4), hip.DevBuf(M * O * 2 + 256)
    w = rng.integers(-128, 128, (O, K), dtype=np.int8)
    dw, dsw = hip.DevBuf.from_array(w), hip.DevBuf.from_array(np.ones(O, np.float32))
    hip._check(L.apus_hip_memset(da.ptr, 2, M * K), "memset")
    hip._check(L.apus_hip_memset(ds.ptr, 0x3F, M * 4), "memset")
    hip._check(L.apus_hip_memset(do.ptr + M * O * 2, 0xA5, 256), "memset")
    sa = np.full(n, np.uint32(0x3F3F3F3F)).view(np.float32)
    tail = rng.integers(-128, 128, (n, K), dtype=np.int8)
    places = (0, M // 2 + 1, M - n)
    for at in places:
        hip._check(L.apus_hip_h2d(da.ptr + at * K, tail.ctypes.data, tail.nbytes), "h2d")
    hip._check(L.apus_hip_i8_gemm_dev(dw.ptr, dsw.ptr, da.ptr, ds.ptr, do.ptr, M, O, K, hip.Y_BF16), "i8_gemm")
    hip.synchronize()
    got = np.empty((n, O), np.uint16)
    for at in places + (5000, M - 5000):
        a = tail if at in places else np.full((n, K), 2, np.int8)
        hip._check(L.apus_hip_d2h(got.ctypes.data, do.ptr + at * O * 2, got.nbytes), "d2h")
        assert np.array_equal(got, R.bf16_bits(R.product(a, sa, w, np.ones(O))))
    end = np.empty(256, np.uint8)
    hip._check(L.apus_hip_d2h(end.ctypes.data, do.ptr + M * O * 2, 256), "d2h")
    assert (end == 0xA5).all()


def test_i8_linear_of_the_most_channels(hip, rng):
    """2^26 channels of more than 2048 elements: a workgroup more than one row's schedule may have,
    for codes and for activations quantised in the call"""
    L = hip.lib()
    O, K, n = 1 << 26, 2064, 40
    dw, one = hip.DevBuf(O * K), hip.DevBuf(O * 4)
    hip._check(L.apus_hip_memset(dw.ptr, 3, O * K), "memset")
    hip._check(L.apus_hip_memset(one.ptr, 0x3F, O * 4), "memset")
    tail = rng.integers(-128, 128, (n, K), dtype=np.int8)
    hip._check(L.apus_hip_h2d(dw.ptr + (O - n) * K, tail.ctypes.data, tail.nbytes), "h2d")
    x = rng.standard_normal((1, K)).astype(np.float32)
    a, sa = R.quant_i8(R.round_bf16(x))
    dx, da, dsa, do = (hip.DevBuf.from_array(v) for v in (x, a, sa, np.zeros(O, np.float32)))
    ws = hip.DevBuf(L.apus_hip_i8_linear_workspace(1, K))
    sw = np.full(n, np.uint32(0x3F3F3F3F)).view(np.float32)
    got = np.empty(n, np.float32)
    for linear in (False, True):
        hip._check(L.apus_hip_memset(do.ptr, 0, O * 4), "memset")
        if linear:
            hip._check(L.apus_hip_i8_linear_dev(dw.ptr, one.ptr, dx.ptr, do.ptr, 1, K, O, 0, ws.ptr), "i8_linear")
        else:
            hip._check(L.apus_hip_i8_gemm_dev(dw.ptr, one.ptr, da.ptr, dsa.ptr, do.ptr, 1, O, K, 0), "i8_gemm")
        hip.synchronize()
        for at, w in ((0, np.full((n, K), 3, np.int8)), (O - n, tail)):
            hip._check(L.apus_hip_d2h(got.ctypes.data, do.ptr + at * 4, got.nbytes), "d2h")
            assert np.array_equal(got, R.product(a, sa, w, sw)[0])
