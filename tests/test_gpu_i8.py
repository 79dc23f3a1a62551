"""apus_hip_i8_gemm_dev and apus_hip_i8_linear_dev: the integer sum is exact and
every rounding after it is documented, so outputs are compared bit for bit."""
import numpy as np
import pytest

import rowops as R

pytestmark = pytest.mark.gpu


def operands(rng, M, O, K):
    a = rng.integers(-128, 128, (M, K), dtype=np.int8)
    w = rng.integers(-128, 128, (O, K), dtype=np.int8)
    sa = (rng.random(M) * 0.1 + 1e-3).astype(np.float32)
    sw = (rng.random(O) * 0.01 + 1e-4).astype(np.float32)
    return a, sa, w, sw


def at(hip, raw, off):
    """a device copy of raw that starts off bytes into its buffer"""
    b = hip.DevBuf.from_array(np.concatenate([np.zeros(off, np.uint8), np.ascontiguousarray(raw).view(np.uint8).ravel()]))
    return b, b.ptr + off


def finish(want, flags, hip):
    if flags & hip.Y_BF16:
        return R.bf16_bits(want)
    return R.round_bf16(want) if flags & hip.R_OUT else want


def gemm(hip, a, sa, w, sw, flags=0, offs=(0, 0, 0)):
    (M, K), O = a.shape, w.shape[0]
    e = 2 if flags & hip.Y_BF16 else 4
    (bw, pw), (ba, pa) = at(hip, w, offs[0]), at(hip, a, offs[1])
    bo, po = at(hip, np.full(M * O * e + 256, 0xA5, np.uint8), offs[2])
    ds, dw = hip.DevBuf.from_array(sa), hip.DevBuf.from_array(sw)
    hip._check(hip.lib().apus_hip_i8_gemm_dev(pw, dw.ptr, pa, ds.ptr, po, M, O, K, flags), "i8_gemm")
    raw = bo.to_array(np.uint8, (offs[2] + M * O * e + 256,))
    assert (raw[:offs[2]] == 0).all() and (raw[offs[2] + M * O * e:] == 0xA5).all()
    return raw[offs[2]:offs[2] + M * O * e].copy().view(np.uint16 if e == 2 else np.float32).reshape(M, O)


def check(hip, rng, M, O, K, flags=0, offs=(0, 0, 0)):
    a, sa, w, sw = operands(rng, M, O, K)
    got = gemm(hip, a, sa, w, sw, flags, offs)
    assert np.array_equal(got, finish(R.product(a, sa, w, sw), flags, hip)), (M, O, K, flags, offs)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 257])
@pytest.mark.parametrize("O,K", [(128, 256), (256, 1024), (200, 512), (33, 2048)])
def test_i8_rows(hip, rng, M, O, K):
    check(hip, rng, M, O, K, hip.Y_BF16 if M % 2 else 0)


@pytest.mark.parametrize("K", [4, 8, 12, 16, 20, 32, 48, 60, 64, 80, 112, 128, 144, 192, 240, 256, 272, 384, 496, 1000, 1008,
                               1024, 1040, 1536, 2064, 4096, 4112, 8192])
@pytest.mark.parametrize("M,O", [(1, 130), (6, 64), (21, 100), (70, 150), (150, 260)])
def test_i8_lengths(hip, rng, K, M, O):
    check(hip, rng, M, O, K)


@pytest.mark.parametrize("O", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 255, 257, 1000, 4097])
@pytest.mark.parametrize("M", [1, 3, 12, 40, 140])
def test_i8_channels(hip, rng, O, M):
    check(hip, rng, M, O, 320, hip.Y_BF16)
    check(hip, rng, M, O, 320, hip.R_OUT)


@pytest.mark.parametrize("M,O,K", [(512, 1024, 1024), (1000, 1000, 2048), (300, 2048, 4096), (1025, 640, 512),
                                   (256, 4096, 128), (2048, 256, 256), (700, 3000, 1040)])
@pytest.mark.parametrize("bf", [False, True])
def test_i8_many_rows(hip, rng, M, O, K, bf):
    check(hip, rng, M, O, K, hip.Y_BF16 if bf else 0)


@pytest.mark.parametrize("M,O", [(777, 4225), (8205, 131), (1671, 1414), (8445, 401), (8300, 70)])
@pytest.mark.parametrize("K", [16, 112, 128, 144, 256, 272, 400, 512, 560, 656, 1152])
def test_i8_ragged_tiles(hip, rng, M, O, K):
    """more and fewer steps of K than a tile's loads under way, whole and ragged last steps,
    rows and channels that end inside a tile, of each tile size"""
    check(hip, rng, M, O, K, hip.Y_BF16 if K % 3 else 0)


@pytest.mark.parametrize("M,O,K", [(2690, 4369, 112), (1420, 8231, 496), (775, 9381, 1072), (1675, 6933, 640)])
def test_i8_ragged_largest_tiles(hip, rng, M, O, K):
    check(hip, rng, M, O, K, 0 if K % 128 else hip.Y_BF16)


@pytest.mark.parametrize("offs", [(4, 0, 0), (0, 4, 0), (0, 0, 4), (8, 8, 8), (12, 4, 12)])
@pytest.mark.parametrize("M", [1, 5, 20, 200])
def test_i8_alignment(hip, rng, offs, M):
    check(hip, rng, M, 192, 256, 0, offs)
    check(hip, rng, M, 192, 256, hip.Y_BF16, offs)
    check(hip, rng, M, 191, 256, hip.Y_BF16, (offs[0], offs[1], 2))


@pytest.mark.parametrize("M", [1, 4, 16, 130])
def test_i8_extreme_sums(hip, M):
    """the largest sums: -128 * -128 * K at the largest K, and its negative"""
    K, O = 131056, 64
    a = np.full((M, K), -128, np.int8)
    w = np.full((O, K), -128, np.int8)
    w[1::2] = 127
    one = np.ones(max(M, O), np.float32)
    got = gemm(hip, a, one[:M], w, one[:O])
    assert np.array_equal(got, R.product(a, one[:M], w, one[:O]))
    assert got[0, 0] == np.float32(2147221504.0)


def test_i8_scales(hip, rng):
    """a NaN scale makes its row NaN, the others stay; zero and infinite scales as multiplied"""
    a, sa, w, sw = operands(rng, 9, 70, 256)
    clean = gemm(hip, a, sa, w, sw)
    sa = sa.copy()
    sa[3], sa[5] = np.nan, 0.0
    got = gemm(hip, a, sa, w, sw)
    keep = [0, 1, 2, 4, 6, 7, 8]
    assert np.array_equal(got[keep], clean[keep]) and np.isnan(got[3]).all() and not got[5].any()
    assert np.isnan(R.from_bf16(gemm(hip, a, sa, w, sw, hip.Y_BF16)[3])).all()


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16, 33, 130])
@pytest.mark.parametrize("O,K", [(128, 256), (100, 1024), (257, 400), (64, 4096), (48, 8192), (32, 100)])
@pytest.mark.parametrize("bf", [False, True])
def test_i8_linear(hip, rng, M, O, K, bf):
    x = (rng.standard_normal((M, K)) * np.exp(2 * rng.standard_normal((M, 1)))).astype(np.float32)
    if M > 2:
        x[1] = 0.0
    _, _, w, sw = operands(rng, 1, O, K)
    b = R.round_bf16(x)
    q, s = R.quant_i8(b)
    dx = hip.DevBuf.from_array(R.bf16_bits(x) if bf else x)
    dw, dsw = hip.DevBuf.from_array(w), hip.DevBuf.from_array(sw)
    L = hip.lib()
    ws = hip.DevBuf(L.apus_hip_i8_linear_workspace(M, K))
    for flags in (0, hip.R_OUT, hip.Y_BF16):
        e = 2 if flags & hip.Y_BF16 else 4
        do = hip.DevBuf.from_array(np.full(M * O * e + 64, 0xA5, np.uint8))
        hip._check(L.apus_hip_i8_linear_dev(dw.ptr, dsw.ptr, dx.ptr, do.ptr, M, K, O, flags | (hip.X_BF16 if bf else 0),
                                            ws.ptr), "i8_linear")
        raw = do.to_array(np.uint8, (M * O * e + 64,))
        assert (raw[M * O * e:] == 0xA5).all()
        got = raw[:M * O * e].copy().view(np.uint16 if e == 2 else np.float32).reshape(M, O)
        assert np.array_equal(got, finish(R.product(q, s, w, sw), flags, hip))


@pytest.mark.parametrize("M", [1, 3, 20])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_i8_linear_non_finite_row(hip, rng, M, value):
    K, O = 512, 96
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[M - 1, 77] = value
    _, _, w, sw = operands(rng, 1, O, K)
    dx, dw, dsw = (hip.DevBuf.from_array(v) for v in (x, w, sw))
    L = hip.lib()
    ws, do = hip.DevBuf(L.apus_hip_i8_linear_workspace(M, K)), hip.DevBuf(M * O * 4)
    hip._check(L.apus_hip_i8_linear_dev(dw.ptr, dsw.ptr, dx.ptr, do.ptr, M, K, O, 0, ws.ptr), "i8_linear")
    got = do.to_array(np.float32, (M, O))
    assert np.isnan(got[M - 1]).all() and np.isfinite(got[:M - 1]).all()


def test_i8_rows_past_32_bits(hip, rng):
    """activation and output offsets that pass 2^32"""
    L = hip.lib()
    for M, O, K in ((1048600, 64, 4096), (70000, 65536, 32)):
        da, dw = hip.DevBuf(M * K), hip.DevBuf.from_array(rng.integers(-128, 128, (O, K), dtype=np.int8))
        hip._check(L.apus_hip_memset(da.ptr, 1, M * K), "memset")
        tail = rng.integers(-128, 128, (3, K), dtype=np.int8)
        hip._check(L.apus_hip_h2d(da.ptr + (M - 3) * K, tail.ctypes.data, 3 * K), "h2d")
        ds, dsw = hip.DevBuf.from_array(np.ones(M, np.float32)), hip.DevBuf.from_array(np.ones(O, np.float32))
        do = hip.DevBuf(M * O * 2)
        hip._check(L.apus_hip_i8_gemm_dev(dw.ptr, dsw.ptr, da.ptr, ds.ptr, do.ptr, M, O, K, hip.Y_BF16), "i8_gemm")
        hip.synchronize()
        got = np.empty((4, O), np.uint16)
        hip._check(L.apus_hip_d2h(got.ctypes.data, do.ptr + (M - 4) * O * 2, got.nbytes), "d2h")
        w = dw.to_array(np.int8, (O, K))
        a = np.concatenate([np.ones((1, K), np.int8), tail])
        assert np.array_equal(got, R.bf16_bits(R.product(a, np.ones(4), w, np.ones(O))))


def test_i8_more_channels_than_workgroups(hip, rng):
    """one row and 2^26 + 5 channels: the outputs at both ends"""
    L = hip.lib()
    O, K = (1 << 26) + 5, 16
    dw, da = hip.DevBuf(O * K), hip.DevBuf.from_array(rng.integers(-128, 128, (1, K), dtype=np.int8))
    hip._check(L.apus_hip_memset(dw.ptr, 3, O * K), "memset")
    tail = rng.integers(-128, 128, (7, K), dtype=np.int8)
    hip._check(L.apus_hip_h2d(dw.ptr + (O - 7) * K, tail.ctypes.data, tail.nbytes), "h2d")
    one = hip.DevBuf.from_array(np.ones(O, np.float32))
    do = hip.DevBuf(O * 4)
    hip._check(L.apus_hip_i8_gemm_dev(dw.ptr, one.ptr, da.ptr, one.ptr, do.ptr, 1, O, K, 0), "i8_gemm")
    hip.synchronize()
    a = da.to_array(np.int8, (1, K))
    w = np.concatenate([np.full((5, K), 3, np.int8), tail])
    want = R.product(a, np.ones(1), w, np.ones(len(w)))[0]
    head, end = np.empty(5, np.float32), np.empty(7, np.float32)
    hip._check(L.apus_hip_d2h(head.ctypes.data, do.ptr, head.nbytes), "d2h")
    hip._check(L.apus_hip_d2h(end.ctypes.data, do.ptr + (O - 7) * 4, end.nbytes), "d2h")
    assert np.array_equal(head, want[:5]) and np.array_equal(end, want[5:])
