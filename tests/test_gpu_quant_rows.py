"""apus_hip_i8_quant_dev at the largest number of rows: a row's number and ROWS_MAX more pass 2^31."""
import numpy as np
import pytest

import rowops as R

pytestmark = pytest.mark.gpu


def test_i8_quant_most_rows(hip):
    """2^31 - 256 rows of one element, all zero but for three places; the rows behind a wrapped
    number would be far in front of the arrays"""
    M, N = 0x7FFFFF00, 1000
    L = hip.lib()
    x, codes, scales = hip.DevBuf(2 * M), hip.DevBuf(M + 256), hip.DevBuf(4 * M + 256)
    hip._check(L.apus_hip_memset(x.ptr, 0, 2 * M), "memset")
    hip._check(L.apus_hip_memset(codes.ptr, 0xA5, M + 256), "memset")
    hip._check(L.apus_hip_memset(scales.ptr, 0xA5, 4 * M + 256), "memset")
    places = (0, (1 << 31) - (1 << 20) - N // 2, M - N)
    v = np.random.default_rng(3).standard_normal((len(places), N, 1)).astype(np.float32)
    raw = R.bf16_bits(v)
    for at, r in zip(places, raw):
        hip._check(L.apus_hip_h2d(x.ptr + 2 * at, r.ctypes.data, r.nbytes), "h2d")
    hip._check(L.apus_hip_i8_quant_dev(x.ptr, M, 1, hip.X_BF16, codes.ptr, scales.ptr), "i8_quant")
    hip.synchronize()
    c, s = np.empty(N, np.int8), np.empty(N, np.float32)
    for at, r in zip(places, v):
        hip._check(L.apus_hip_d2h(c.ctypes.data, codes.ptr + at, c.nbytes), "d2h")
        hip._check(L.apus_hip_d2h(s.ctypes.data, scales.ptr + 4 * at, s.nbytes), "d2h")
        wc, ws = R.quant_i8(R.round_bf16(r))
        assert np.array_equal(c, wc[:, 0]) and np.array_equal(s, ws)
    wc, ws = R.quant_i8(np.zeros((1, 1), np.float32))
    for at in (N, 1 << 30, (1 << 31) - (1 << 19), M - 2 * N):            # rows of zeros between them
        hip._check(L.apus_hip_d2h(c.ctypes.data, codes.ptr + at, c.nbytes), "d2h")
        hip._check(L.apus_hip_d2h(s.ctypes.data, scales.ptr + 4 * at, s.nbytes), "d2h")
        assert not c.any() and (s == ws[0]).all()
    tail = np.empty(256, np.uint8)
    for b, n in ((codes, M), (scales, 4 * M)):
        hip._check(L.apus_hip_d2h(tail.ctypes.data, b.ptr + n, 256), "d2h")
        assert (tail == 0xA5).all()
