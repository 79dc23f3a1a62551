"""apus_hip_rmsnorm_dev and apus_hip_i8_quant_dev against the 64-bit formulas.

Tolerances: the device's 64-bit value is within a few 2^-53 (a sum of K <= 2^15
squares in any order: 2^-37 at most, half of that in y) of the formula's, then
rounded once to fp32 (half a step, 2^-24) and to BF16 (2^-8). The residual's sum
is one fp32 addition (and a BF16 rounding): bitwise. Codes and scales are made of
bf16(y): bitwise equal to the act quant's (the oracle) or the integer rule applied
to the y that the same call returns."""
import numpy as np
import pytest

import rowops as R

pytestmark = pytest.mark.gpu

EPS = 1e-6
F32, BF = 2.0 ** -24 + 2.0 ** -36, 2.0 ** -8 + 2.0 ** -23


def dev(hip, a):
    return hip.DevBuf.from_array(a)


def store(v, bf):
    return R.bf16_bits(v) if bf else np.ascontiguousarray(v, np.float32)


def fetch(buf, bf, shape):
    return R.from_bf16(buf.to_array(np.uint16, shape)) if bf else buf.to_array(np.float32, shape)


def guarded(hip, nbytes):
    """a buffer of nbytes with 256 guard bytes behind it, all 0xA5"""
    return dev(hip, np.full(nbytes + 256, 0xA5, np.uint8))


def check_guard(buf, nbytes):
    assert (buf.to_array(np.uint8, (nbytes + 256,))[nbytes:] == 0xA5).all()


def run(hip, oracle, x, res, gamma, quant, xb, yb, ldx=None, gb=False, r_out=False, shift=0, want_y=True, check=True):
    M, K = x.shape
    ldx = ldx or K
    wide = np.full((M, ldx), 7.0, np.float32)
    wide[:, :K] = x
    ex, ey = 2 if xb else 4, 2 if yb else 4
    raw = store(wide, xb)
    # shift: the rows start that many elements into the buffer
    dx = dev(hip, np.concatenate([np.zeros(shift, raw.dtype), raw.ravel()]))
    dr = dev(hip, store(res, xb)) if res is not None else None
    dg = dev(hip, store(gamma, gb))
    do = guarded(hip, M * K * ex) if res is not None else None
    dy = guarded(hip, M * K * ey) if want_y else None
    dc = guarded(hip, M * K) if quant else None
    ns = 0 if not quant else M * (K // 128) if quant == "e4m3" else M
    ds = guarded(hip, ns * 4) if quant else None
    flags = ((hip.X_BF16 if xb else 0) | (hip.Y_BF16 if yb else 0) | (hip.W_BF16 if gb else 0) |
             (hip.R_OUT if r_out else 0) | (hip.Q_I8 if quant == "i8" else 0))
    p = lambda b: b.ptr if b is not None else None  # noqa: E731
    hip._check(hip.lib().apus_hip_rmsnorm_dev(dx.ptr + shift * ex, ldx, p(dr), p(do), dg.ptr, M, K, EPS, flags, p(dy),
                                              p(dc), p(ds)), "rmsnorm")
    hip.synchronize()
    out = {}
    xs = fetch(dx, xb, (shift + M * ldx,))[shift:].reshape(M, ldx)[:, :K]
    r = xs
    if res is not None:
        with np.errstate(invalid="ignore", over="ignore"):
            r = xs + fetch(dr, xb, (M, K))
        r = R.round_bf16(r) if xb else r
        out["r"] = fetch(do, xb, (M, K))
        check_guard(do, M * K * ex)
        if check:
            assert np.array_equal(out["r"].view(np.uint32), r.view(np.uint32))
    g = R.from_bf16(store(gamma, True)) if gb else gamma.astype(np.float32)
    truth = R.norm_truth(r, g, EPS)
    if want_y:
        out["y"] = fetch(dy, yb, (M, K))
        check_guard(dy, M * K * ey)
        if check:
            tol = (BF if yb or r_out else F32) * np.abs(truth) + 1e-44
            assert (np.abs(out["y"] - truth) <= tol).all(), np.abs(out["y"] / truth - 1).max()
            if r_out and not yb:
                assert np.array_equal(R.round_bf16(out["y"]), out["y"])
    if quant:
        shape = (M, K // 128) if quant == "e4m3" else (M,)
        out["codes"] = dc.to_array(np.uint8, (M, K)).view(np.int8 if quant == "i8" else np.uint8)
        out["scales"] = ds.to_array(np.float32, (ns,)).reshape(shape)
        check_guard(dc, M * K)
        check_guard(ds, ns * 4)
        if check and want_y:
            b = R.round_bf16(out["y"])
            codes, scales = R.quant_i8(b) if quant == "i8" else R.quant_e4m3(oracle, b)
            assert np.array_equal(out["scales"], scales)
            assert np.array_equal(out["codes"], codes)
    return out


def inputs(rng, M, K, res):
    x = (rng.standard_normal((M, K)) * np.exp(rng.standard_normal((1, K)))).astype(np.float32)
    return x, (3 * rng.standard_normal((M, K))).astype(np.float32) if res else None, \
        (1 + 0.3 * rng.standard_normal(K)).astype(np.float32)


@pytest.mark.parametrize("K", [128, 384, 512, 1024, 1536, 2048, 4096, 5120, 8192, 16384, 20480])
@pytest.mark.parametrize("quant", ["e4m3", "i8", None])
@pytest.mark.parametrize("xb,yb", [(False, False), (True, True), (True, False), (False, True)])
def test_norm_lengths(hip, oracle, rng, K, quant, xb, yb):
    M = 5 if K < 8192 else 2
    x, res, gamma = inputs(rng, M, K, True)
    run(hip, oracle, x, res, gamma, quant, xb, yb)


@pytest.mark.parametrize("K", [1, 2, 7, 63, 100, 1000, 1001, 4100, 8200])
@pytest.mark.parametrize("quant", ["i8", None])
@pytest.mark.parametrize("bf", [False, True])
def test_norm_odd_lengths(hip, oracle, rng, K, quant, bf):
    x, res, gamma = inputs(rng, 3, K, True)
    run(hip, oracle, x, res, gamma, quant, bf, bf)
    run(hip, oracle, x, None, gamma, quant, bf, bf)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 7, 8, 9, 64, 255, 1025])
@pytest.mark.parametrize("quant", ["e4m3", "i8"])
def test_norm_rows(hip, oracle, rng, M, quant):
    x, res, gamma = inputs(rng, M, 1024, True)
    run(hip, oracle, x, res, gamma, quant, True, True)


@pytest.mark.parametrize("K,ldx,shift", [(1024, 1536, 0), (512, 1536, 1024), (1024, 1029, 0), (1024, 1024, 1),
                                         (1024, 1032, 4), (256, 260, 2), (4096, 4099, 3)])
@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("quant", ["e4m3", "i8"])
def test_norm_strided_and_misaligned_rows(hip, oracle, rng, K, ldx, shift, bf, quant):
    x, _, gamma = inputs(rng, 6, K, False)
    run(hip, oracle, x, None, gamma, quant, bf, bf, ldx=ldx, shift=shift)


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("quant", ["e4m3", "i8"])
def test_norm_outputs_do_not_depend_on_each_other(hip, oracle, rng, bf, quant):
    """the same codes with and without y, and y with and without codes"""
    x, res, gamma = inputs(rng, 4, 1280, True)
    a = run(hip, oracle, x, res, gamma, quant, bf, bf)
    b = run(hip, oracle, x, res, gamma, quant, bf, bf, want_y=False)
    c = run(hip, oracle, x, res, gamma, None, bf, bf)
    for k in ("codes", "scales"):
        assert np.array_equal(a[k], b[k])
    assert np.array_equal(a["y"], c["y"])


def test_norm_flags(hip, oracle, rng):
    """BF16 gamma, BF16-rounded fp32 y"""
    x, res, gamma = inputs(rng, 5, 640, True)
    run(hip, oracle, x, res, gamma, "e4m3", False, False, gb=True, r_out=True)
    run(hip, oracle, x, res, gamma, "i8", True, False, gb=True, r_out=True)
    run(hip, oracle, x[:, :77], res[:, :77], gamma[:77], "i8", True, True, gb=True)


def test_norm_codes_independent_of_the_batch(hip, oracle, rng):
    x, res, gamma = inputs(rng, 300, 2048, True)
    for quant in ("e4m3", "i8"):
        a = run(hip, oracle, x, res, gamma, quant, True, True, check=False)
        b = run(hip, oracle, x[17:18], res[17:18], gamma, quant, True, True)
        for k in ("r", "y", "codes", "scales"):
            assert np.array_equal(a[k][17:18], b[k])


@pytest.mark.parametrize("K", [256, 4096, 260])
@pytest.mark.parametrize("bf", [False, True])
def test_norm_zero_tiny_and_huge_rows(hip, oracle, K, bf):
    x = np.zeros((6, K), np.float32)
    x[1] = 1e-30
    x[2, 3] = 1e-38
    x[3] = 3e38 * np.where(np.arange(K) % 2, 1, -1)
    x[4, K - 1] = -3e38
    x[5, ::5] = 1e-3
    gamma = np.ones(K, np.float32)
    run(hip, oracle, x, None, gamma, "i8", bf, bf)
    if K % 128 == 0:
        run(hip, oracle, x, None, gamma, "e4m3", bf, bf)
    run(hip, oracle, x, None, np.zeros(K, np.float32), "i8", bf, bf)


@pytest.mark.parametrize("K", [256, 4096, 260])
@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_norm_non_finite_row_stays_alone(hip, oracle, rng, K, bf, value):
    x, res, gamma = inputs(rng, 4, K, True)
    clean = {q: run(hip, oracle, x, res, gamma, q, bf, bf) for q in ("i8", "e4m3") if q == "i8" or K % 128 == 0}
    x = x.copy()
    x[2, K // 2] = value
    for q, c in clean.items():
        o = run(hip, oracle, x, res, gamma, q, bf, bf, check=False)
        rows = [0, 1, 3]
        for k in ("y", "codes", "scales"):
            assert np.array_equal(o[k][rows], c[k][rows])
        assert not o["codes"][2].any()
        assert np.isnan(o["scales"][2]).all() if q == "i8" else np.isposinf(o["scales"][2]).all()
        y = o["y"][2]
        if np.isnan(value):
            assert np.isnan(y).all()
        else:
            assert np.isnan(y[K // 2]) and not np.delete(y, K // 2).any()


@pytest.mark.parametrize("quant", ["e4m3", "i8", None])
@pytest.mark.parametrize("K", [1024, 640, 40960])
def test_norm_in_place(hip, oracle, rng, quant, K):
    """res_out over res, y over x; res_out over x, y over res"""
    M = 3
    x, res, gamma = inputs(rng, M, K, True)
    want = run(hip, oracle, x, res, gamma, quant, False, False)
    for swap in (False, True):
        dx, dr, dg = dev(hip, x), dev(hip, res), dev(hip, gamma)
        dc, ds = hip.DevBuf(M * K), hip.DevBuf(M * K)
        o, y = (dx, dr) if swap else (dr, dx)
        hip._check(hip.lib().apus_hip_rmsnorm_dev(dx.ptr, K, dr.ptr, o.ptr, dg.ptr, M, K, EPS,
                                                  hip.Q_I8 if quant == "i8" else 0, y.ptr, dc.ptr if quant else None,
                                                  ds.ptr if quant else None), "rmsnorm")
        assert np.array_equal(o.to_array(np.float32, (M, K)), want["r"])
        assert np.array_equal(y.to_array(np.float32, (M, K)), want["y"])
        if quant:
            assert np.array_equal(dc.to_array(np.uint8, (M, K)).view(want["codes"].dtype), want["codes"])
    # y over x without res_out
    dx, dr, dg = dev(hip, x), dev(hip, res), dev(hip, gamma)
    hip._check(hip.lib().apus_hip_rmsnorm_dev(dx.ptr, K, dr.ptr, None, dg.ptr, M, K, EPS, 0, dx.ptr, None, None), "rmsnorm")
    assert np.array_equal(dx.to_array(np.float32, (M, K)), want["y"])


def test_norm_only_the_residual(hip, rng):
    x, res, gamma = inputs(rng, 3, 512, True)
    dx, dr, dg = dev(hip, x), dev(hip, res), dev(hip, gamma)
    hip._check(hip.lib().apus_hip_rmsnorm_dev(dx.ptr, 512, dr.ptr, dr.ptr, dg.ptr, 3, 512, EPS, 0, None, None, None), "rmsnorm")
    assert np.array_equal(dr.to_array(np.float32, (3, 512)), x + res)


def test_norm_rows_past_32_bits(hip):
    """the last rows of arrays whose offsets pass 2^32 elements"""
    K, M = 65536, 65540
    x, codes, scales = hip.DevBuf(M * K * 2), hip.DevBuf(M * K), hip.DevBuf(M * 4)
    L = hip.lib()
    g = dev(hip, np.ones(K, np.float32))
    rng = np.random.default_rng(5)
    tail = (rng.standard_normal((3, K))).astype(np.float32)
    hip._check(L.apus_hip_memset(x.ptr, 0, M * K * 2), "memset")
    raw = R.bf16_bits(tail)
    hip._check(L.apus_hip_h2d(x.ptr + (M - 3) * K * 2, raw.ctypes.data, raw.nbytes), "h2d")
    hip._check(L.apus_hip_rmsnorm_dev(x.ptr, K, None, None, g.ptr, M, K, EPS, hip.X_BF16 | hip.Q_I8, None, codes.ptr,
                                      scales.ptr), "rmsnorm")
    hip.synchronize()
    got = np.empty((3, K), np.int8)
    hip._check(L.apus_hip_d2h(got.ctypes.data, codes.ptr + (M - 3) * K, 3 * K), "d2h")
    y = R.norm_truth(R.round_bf16(tail), np.ones(K, np.float32), EPS).astype(np.float32)
    want, ws = R.quant_i8(R.round_bf16(y))
    s = scales.to_array(np.float32, (M,))
    assert np.array_equal(s[-3:], ws) and (s[:5] == s[0]).all()
    # y may round the other way where its 64-bit value lies within 2^-36 of a border
    assert np.mean(got != want) < 1e-5 and np.abs(got.astype(int) - want).max() <= 1


# ------------------------------------------------------------ integer quantiser


@pytest.mark.parametrize("M,K", [(1, 1), (3, 5), (1, 4096), (37, 1024), (5, 1000), (2, 8192), (3, 20000), (300, 64), (9, 1001)])
@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_i8_quant(hip, rng, M, K, bf, shift):
    x = (rng.standard_normal((M, K)) * np.exp(3 * rng.standard_normal((M, 1)))).astype(np.float32)
    if M > 2:
        x[1] = 0
        x[2] *= np.float32(1e-37)
    raw = store(x, bf)
    dx = dev(hip, np.concatenate([np.zeros(shift, raw.dtype), raw.ravel()]))
    dc, ds = guarded(hip, M * K), guarded(hip, M * 4)
    hip._check(hip.lib().apus_hip_i8_quant_dev(dx.ptr + shift * raw.itemsize, M, K, hip.X_BF16 if bf else 0, dc.ptr,
                                               ds.ptr), "i8_quant")
    hip.synchronize()
    codes, scales = R.quant_i8(R.round_bf16(x))
    assert np.array_equal(ds.to_array(np.float32, (M,)), scales)
    assert np.array_equal(dc.to_array(np.int8, (M, K)), codes)
    check_guard(dc, M * K)
    check_guard(ds, M * 4)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("K", [256, 1001])
def test_i8_quant_non_finite_row(hip, rng, value, K):
    x = rng.standard_normal((3, K)).astype(np.float32)
    x[1, K - 1] = value
    dx, dc, ds = dev(hip, x), hip.DevBuf(3 * K), hip.DevBuf(12)
    hip._check(hip.lib().apus_hip_i8_quant_dev(dx.ptr, 3, K, 0, dc.ptr, ds.ptr), "i8_quant")
    codes, s = dc.to_array(np.int8, (3, K)), ds.to_array(np.float32, (3,))
    want, ws = R.quant_i8(R.round_bf16(x[[0, 2]]))
    assert np.array_equal(codes[[0, 2]], want) and np.array_equal(s[[0, 2]], ws)
    assert not codes[1].any() and np.isnan(s[1])


def test_rows_in_more_than_one_round(hip, oracle, rng):
    """more rows than a launch has workgroups for"""
    M, K = (1 << 20) + 77, 16
    base = rng.standard_normal((64, K)).astype(np.float32)
    x = np.tile(base, (M // 64 + 1, 1))[:M]
    gamma = (1 + 0.3 * rng.standard_normal(K)).astype(np.float32)
    want = run(hip, oracle, base, None, gamma, "i8", False, False)
    dx, dg = dev(hip, x), dev(hip, gamma)
    dc, ds = hip.DevBuf(M * K), hip.DevBuf(M * 4)
    L = hip.lib()
    r = np.arange(M) % 64
    hip._check(L.apus_hip_rmsnorm_dev(dx.ptr, K, None, None, dg.ptr, M, K, EPS, hip.Q_I8, None, dc.ptr, ds.ptr), "norm")
    assert np.array_equal(dc.to_array(np.int8, (M, K)), want["codes"][r])
    assert np.array_equal(ds.to_array(np.float32, (M,)), want["scales"][r])
    for k in (K, 4):                             # 4: the kernel of short rows
        hip._check(L.apus_hip_i8_quant_dev(dx.ptr, M, k, 0, dc.ptr, ds.ptr), "quant")
        pieces = base.reshape(-1, k)
        codes, scales = R.quant_i8(R.round_bf16(pieces))
        at = np.arange(M) % len(pieces)
        assert np.array_equal(dc.to_array(np.int8, (M, k)), codes[at])
        assert np.array_equal(ds.to_array(np.float32, (M,)), scales[at])


@pytest.mark.parametrize("K", [8, 9, 15, 44, 120, 127, 128, 129, 136, 200, 255, 256, 257])
@pytest.mark.parametrize("M", [1, 7, 16, 33, 700])
@pytest.mark.parametrize("bf", [False, True])
def test_several_short_rows_a_wave(hip, oracle, rng, K, M, bf):
    """rows that share a wave, the last wave not full; a non-finite row beside the others"""
    for quant in (["e4m3", "i8"] if K % 128 == 0 else ["i8", None]):
        run(hip, oracle, *inputs(rng, M, K, True), quant, bf, bf)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[M // 2, K // 3] = np.nan
    dx, dg = hip.DevBuf.from_array(x), hip.DevBuf.from_array(np.ones(K, np.float32))
    dc, ds = hip.DevBuf(M * K), hip.DevBuf(M * 4)
    L = hip.lib()
    for norm in (True, False):
        if norm:
            hip._check(L.apus_hip_rmsnorm_dev(dx.ptr, K, None, None, dg.ptr, M, K, EPS, hip.Q_I8, None, dc.ptr, ds.ptr), "norm")
        else:
            hip._check(L.apus_hip_i8_quant_dev(dx.ptr, M, K, 0, dc.ptr, ds.ptr), "quant")
        hip.synchronize()
        c, s = dc.to_array(np.int8, (M, K)), ds.to_array(np.float32, (M,))
        bad = np.arange(M) == M // 2
        assert np.isnan(s[bad]).all() and not c[bad].any() and (s[~bad] > 0).all()
        assert (np.abs(c[~bad]).max(1, initial=0) == 127).all()
