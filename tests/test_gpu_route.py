"""apus_hip_route_dev against the 64-bit formulas.

The choice is compared exactly on every token whose deciding values are further
apart than 2^-40 of the largest (the device's exponential and sums are 64-bit to
within a few 2^-53, over at most 2^10 terms), and equal values have to go to the
lowest index. Weights: one rounding to fp32 (half a step, 2^-24) of a 64-bit
value; scores: 2^-21 relative, as documented."""
import ctypes as C

import numpy as np
import pytest

import rowops as R

pytestmark = pytest.mark.gpu

KINDS = {"softplus": 0, "sigmoid": 1, "softmax": 2}


def call(hip, kind, z, bias, topk, groups=1, keep=1, top=1, renorm=1, scale=2.5, want_scores=True, lead=0):
    s, E = z.shape
    zb = np.concatenate([np.zeros(lead, np.float32), z.ravel()])
    dz = hip.DevBuf.from_array(zb)
    db = hip.DevBuf.from_array(bias) if bias is not None else None
    guard = np.full(s * topk * 4 + 64, 0x5A, np.uint8)
    di, dw = hip.DevBuf.from_array(guard), hip.DevBuf.from_array(guard)
    dp = hip.DevBuf.from_array(np.full(s * E * 4 + 64, 0x5A, np.uint8)) if want_scores else None
    cfg = hip.ApusHipRoute(KINDS[kind], topk, groups, keep, top, renorm, scale)
    hip._check(hip.lib().apus_hip_route_dev(C.byref(cfg), dz.ptr + 4 * lead, db.ptr if db else None, s, E, di.ptr,
                                            dw.ptr, dp.ptr if dp else None), "route")
    hip.synchronize()
    for b, n in ((di, s * topk * 4), (dw, s * topk * 4), (dp, s * E * 4)):
        if b:
            assert (b.to_array(np.uint8, (n + 64,))[n:] == 0x5A).all()
    return (di.to_array(np.int32, (s, topk)), dw.to_array(np.float32, (s, topk)),
            dp.to_array(np.float32, (s, E)) if dp else None)


def check(hip, kind, z, bias, topk, groups=1, keep=1, top=1, renorm=1, scale=2.5, lead=0, least=0.95):
    z = z.astype(np.float32)
    idx, wgt, p = call(hip, kind, z, bias, topk, groups, keep, top, renorm, scale, lead=lead)
    wi, ww, wp, gap = R.route(kind, z, bias, topk, groups, keep, top, renorm, scale)
    clear = gap > 2.0 ** -40
    assert clear.mean() > least
    assert np.array_equal(idx[clear], wi[clear])
    assert (np.abs(wgt - ww)[clear] <= (2.0 ** -24 + 2.0 ** -40) * np.abs(ww[clear]) + 2.0 ** -149).all()
    assert (np.abs(p - wp) <= 2.0 ** -21 * wp + 2.0 ** -125).all()
    assert all(len(set(row)) == topk for row in idx.tolist())
    i2, w2, _ = call(hip, kind, z, bias, topk, groups, keep, top, renorm, scale, want_scores=False, lead=lead)
    assert np.array_equal(i2, idx) and np.array_equal(w2, wgt)
    return idx, wgt


def logits(rng, s, E):
    return (1.5 * rng.standard_normal((s, E)) + rng.standard_normal((1, E))).astype(np.float32)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("E,topk", [(1, 1), (2, 1), (7, 3), (8, 8), (16, 16), (60, 4), (64, 6), (65, 2), (128, 8),
                                    (160, 6), (250, 7), (256, 6), (256, 8), (257, 16), (512, 8), (1000, 8), (1024, 16)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_sizes(hip, rng, kind, E, topk, with_bias):
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32) if with_bias else None
    check(hip, kind, logits(rng, 37, E), bias, topk)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("E,groups,keep,topk", [(256, 8, 4, 8), (256, 4, 1, 6), (64, 8, 3, 6), (160, 8, 3, 6), (12, 6, 2, 4),
                                                (256, 64, 16, 8), (256, 16, 16, 8), (96, 3, 2, 5), (1024, 32, 4, 16),
                                                (40, 40, 5, 5), (512, 2, 1, 8), (176, 16, 5, 8), (250, 5, 2, 8)])
@pytest.mark.parametrize("top", [1, 2])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_groups(hip, rng, kind, E, groups, keep, topk, top, with_bias):
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32) if with_bias else None
    check(hip, kind, logits(rng, 29, E), bias, topk, groups, keep, top)


@pytest.mark.parametrize("s", [1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 1000])
def test_route_tokens(hip, rng, s):
    bias = (0.1 * rng.standard_normal(256)).astype(np.float32)
    check(hip, "sigmoid", logits(rng, s, 256), bias, 8, 8, 4, 2)
    check(hip, "softmax", logits(rng, s, 256), None, 6)


@pytest.mark.parametrize("kind", list(KINDS))
def test_route_without_renorm_and_unaligned(hip, rng, kind):
    check(hip, kind, logits(rng, 21, 256), None, 8, renorm=0, scale=1.0)
    check(hip, kind, logits(rng, 21, 255), None, 8, renorm=0, scale=-0.5)
    for lead in (1, 2, 3):
        check(hip, kind, logits(rng, 9, 256), None, 6, lead=lead)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("groups,keep,top", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
def test_route_ties_go_to_the_lowest_index(hip, rng, kind, groups, keep, top):
    """logits on a coarse grid, whole rows equal, equal biases"""
    E = 256
    z = np.round(2 * logits(rng, 40, E)) / 2
    z[3] = 0.25
    z[4] = -5.0
    z[5, ::2] = 1.0
    z[5, 1::2] = 1.0 + 2.0 ** -23            # neighbours in fp32: the larger first
    z[6] = 40.0                              # a sigmoid of 1 for all
    bias = (np.round(4 * rng.standard_normal(E)) / 64).astype(np.float32)
    check(hip, kind, z, None, 8, groups, keep, top)
    check(hip, kind, z, bias, 8, groups, keep, top)
    check(hip, kind, z, np.full(E, -2.0, np.float32), 8, groups, keep, top)


@pytest.mark.parametrize("kind", list(KINDS))
def test_route_scores_next_to_each_other(hip, rng, kind):
    """logits one fp32 step apart: their fp32 scores may be equal, the choice is not"""
    s, E = 64, 128
    base = (0.5 + rng.random((s, 1))).astype(np.float32)
    step = rng.permuted(np.tile(np.arange(E), (s, 1)), axis=1)
    z = (base.view(np.uint32) + step.astype(np.uint32)).view(np.float32)
    check(hip, kind, z, None, 8)
    # a group's sum is a sum of two steps: two of the four groups that decide have equal
    # ones (apart only by the score's curvature, 2^-46) in about one row of six
    check(hip, kind, z, None, 8, 8, 3, 2, least=0.5)
    check(hip, kind, z, (step[0] % 3).astype(np.float32) * np.float32(2.0 ** -24), 8)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("groups,keep,top", [(1, 1, 1), (8, 2, 1), (8, 2, 2)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_masks(hip, rng, kind, groups, keep, top, with_bias):
    E, k = 64, 8
    z = logits(rng, 14, E)
    z[0] = -np.inf                            # nothing left
    z[1] = np.nan
    z[2, 5:] = -np.inf                        # fewer than topk left
    z[3, ::2] = np.nan
    z[4, 8:] = -np.inf                        # one group left
    z[5] = -3.4028235e38                      # lowest value: no mask
    z[6, 1::2] = -3.4028235e38
    z[7, 9] = np.inf
    z[8, [3, 60]] = np.inf
    z[9] = np.inf
    z[10] = 3.4028235e38
    z[11, :63] = -np.inf
    z[12] = -800.0
    bias = None
    if with_bias:
        bias = (0.3 * rng.standard_normal(E)).astype(np.float32)
        bias[[2, 17, 40]] = -np.inf
        bias[50] = np.nan
        bias[33] = np.inf
        bias[7] = -3.4028235e38
    idx, wgt = check(hip, kind, z, bias, k, groups, keep, top)
    assert np.isfinite(wgt).all()
    assert not wgt[0].any() and not wgt[1].any()
    if groups == 1 and not with_bias:
        assert np.array_equal(idx[0], np.arange(k)) and np.array_equal(idx[1], np.arange(k))
        assert set(idx[2, :5]) == set(range(5)) and list(idx[2, 5:]) == [5, 6, 7] and not wgt[2, 5:].any()


def test_route_many_tokens(hip, rng):
    """more tokens than one round of workgroups; the same rows in another order"""
    E, s = 64, 40000
    z = logits(rng, 500, E)
    bias = (0.05 * rng.standard_normal(E)).astype(np.float32)
    pick = rng.integers(0, 500, s)
    a, w, _ = call(hip, "sigmoid", z, bias, 6, 8, 4, 2)
    b, v, _ = call(hip, "sigmoid", z[pick], bias, 6, 8, 4, 2)
    assert np.array_equal(b, a[pick]) and np.array_equal(v, w[pick])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("E,k,groups,keep,top", [(320, 8, 1, 1, 1), (320, 8, 5, 2, 2), (64, 12, 1, 1, 1), (64, 12, 8, 3, 2),
                                                 (512, 8, 16, 4, 1), (1024, 16, 32, 8, 2), (96, 6, 3, 2, 1)])
def test_route_ties_and_masks_other_shapes(hip, rng, kind, E, k, groups, keep, top):
    """many experts, many of them chosen, group counts that do not divide a row of 16 lanes"""
    z = logits(rng, 40, E)
    z[:12] = np.round(2 * z[:12]) / 2
    z[3] = 0.25
    z[4, ::2] = 1.0
    z[4, 1::2] = 1.0 + 2.0 ** -23
    z[12] = -np.inf
    z[13] = np.nan
    z[14, 5:] = -np.inf
    z[15, ::2] = np.nan
    z[16, E // 8:] = -np.inf
    z[17] = -3.4028235e38
    z[18, 1::2] = -3.4028235e38
    z[19, [2, 9, E - 1]] = np.inf
    z[20] = -800.0
    z[21, :E - 1] = -np.inf
    check(hip, kind, z, None, k, groups, keep, top)
    bias = (np.round(4 * rng.standard_normal(E)) / 64).astype(np.float32)
    check(hip, kind, z, bias, k, groups, keep, top)
    bias[[1, 17, 40]] = -np.inf
    bias[50] = np.nan
    bias[33] = np.inf
    idx, wgt = check(hip, kind, z, bias, k, groups, keep, top, renorm=0, scale=1.0)
    assert np.isfinite(wgt).all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("groups,keep,top", [(1, 1, 1), (8, 3, 2), (16, 5, 1)])
@pytest.mark.parametrize("shift,spread", [(-60.0, 3.0), (-20.0, 1.0), (-6.0, 0.01), (0.0, 1e-4), (0.0, 1e-6), (12.0, 0.5),
                                          (60.0, 5.0), (0.0, 40.0), (1e4, 1e3), (-3.0, 1e-3)])
def test_route_where_fp32_tells_little(hip, rng, kind, groups, keep, top, shift, spread):
    """scores that are tiny, saturated or closer than their rounding, with and without a
    bias that swamps or cancels them: the choice stays that of the 64-bit values"""
    E = 256
    z = (shift + spread * rng.standard_normal((24, E))).astype(np.float32)
    check(hip, kind, z, None, 8, groups, keep, top, least=0.0)
    for scale in (1e-6, 1.0, 300.0):
        check(hip, kind, z, (scale * rng.standard_normal(E)).astype(np.float32), 8, groups, keep, top, least=0.0)
    p, _ = R.scores(kind, z[:1])
    check(hip, kind, z, -p[0].astype(np.float32), 8, groups, keep, top, least=0.0)


def test_route_many_tokens_many_experts(hip, rng):
    E, s = 320, 40000
    z = logits(rng, 400, E)
    pick = rng.integers(0, 400, s)
    a, w, _ = call(hip, "softmax", z, None, 8, want_scores=False)
    b, v, _ = call(hip, "softmax", z[pick], None, 8, want_scores=False)
    assert np.array_equal(b, a[pick]) and np.array_equal(v, w[pick])


def test_route_no_tokens(hip):
    cfg = hip.ApusHipRoute(1, 2, 1, 1, 1, 1, 1.0)
    b = hip.DevBuf(64)
    assert hip.lib().apus_hip_route_dev(C.byref(cfg), b.ptr, None, 0, 4, b.ptr + 16, b.ptr + 32, None) == 0
