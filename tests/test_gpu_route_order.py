"""The order of apus_hip_route_dev where fp32 scores of very different size meet: large
scores beside ordinary ones, biases that swamp the scores, groups whose second value is tiny.
The choice has to be that of the 64-bit values (tests/test_gpu_route.py says what is compared)."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_route import KINDS, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,k", [(64, 8), (256, 6), (320, 8), (64, 12)])
@pytest.mark.parametrize("large", [40.0, 2000.0, 1e4, 1e6])
@pytest.mark.parametrize("fine", [0.0, 2.0 ** -22, 2.0 ** -20])
def test_route_large_scores_beside_small_ones(hip, rng, E, k, large, fine):
    """three scores a few fp32 steps apart among ones near 1: sqrt-softplus has no upper end, so
    the largest scores have the largest errors. The bias is a step or so of the large ones."""
    s = 4000
    z = rng.standard_normal((s, E)) - 2.0
    near = large * (1 + rng.integers(0, 64, (s, 3)) * 2.0 ** -23)
    at = np.argsort(rng.random((s, E)), axis=1)[:, :3]
    np.put_along_axis(z, at, near, axis=1)
    bias = (fine * np.sqrt(large) * rng.standard_normal(E)).astype(np.float32) if fine else None
    check(hip, "softplus", z, bias, k, least=0.5)


@pytest.mark.parametrize("E,k", [(64, 8), (256, 6), (320, 8), (64, 12)])
@pytest.mark.parametrize("power", [14, 15, 17])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_route_biases_that_swamp_small_scores(hip, rng, E, k, power, sign):
    """sums in which one step of fp32 is wider than the error of the scores. k experts have a
    bias one step above the others' and a score just over half a step, k more a score just over
    one and a half: less by 64-bit values, but a softplus near zero is known to 2^-24 only, and
    fp32 sums of the former may come out a step below the latter's."""
    s, step = 300, 2.0 ** (power - 23)
    half = step * step / 4                        # the softplus of a score of half a step
    kind = rng.permutation(np.minimum(np.arange(E) // k, 2))
    a = half + 2.0 ** -23 * (0.30 + 0.15 * rng.random((s, E)))
    b = 9 * half + 2.0 ** -23 * (0.55 + 0.10 * rng.random((s, E)))
    z = np.where(kind == 2, -40.0, np.log(np.expm1(np.where(kind == 0, a, b))))
    bias = (sign * 1.5 * 2.0 ** power + step * (kind == 0)).astype(np.float32)
    # the former's scores may lie closer together than 2^-40 of the sums: their set is sure
    idx, _ = check(hip, "softplus", z, bias, k, least=-1.0)
    assert (kind[idx] == 0).all()


@pytest.mark.parametrize("E,groups,keep,k", [(64, 8, 4, 4), (256, 8, 3, 6), (256, 4, 2, 2), (512, 8, 4, 8), (60, 5, 2, 2)])
@pytest.mark.parametrize("first", [0.8, 1.5])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_groups_with_a_tiny_second_value(hip, rng, E, groups, keep, k, first, with_bias):
    """a group's second value may be tiny where its sum is not: a softplus of 0.45 or 0.55 steps
    of 2^-23 comes out as 0 or a whole one, and the groups' largest scores make up for that
    difference in fp32 but not in 64 bits"""
    s, per = 300, E // groups
    low = rng.random((s, groups)) < 0.5
    p1 = first + np.where(low, 1e-4, 0.0) + 1e-6 * rng.random((s, groups))
    second = 2.0 ** -23 * np.where(low, 0.45, 0.55)
    z = np.full((s, groups, per), -30.0) + rng.random((s, groups, per))
    z[:, :, 1] = np.log(np.expm1(p1 * p1))
    z[:, :, per - 1] = np.log(np.expm1(second))
    bias = np.full(E, 0.125, np.float32) if with_bias else None
    check(hip, "softplus", z.reshape(s, E), bias, k, groups, keep, 2, least=0.5)


SHAPES = [(256, 8, 1, 1), (256, 8, 8, 4), (320, 8, 1, 1), (512, 8, 2, 1), (64, 12, 1, 1), (64, 6, 16, 7)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("E,k,groups,keep", SHAPES)
@pytest.mark.parametrize("large", [-1e9, -1e4, 1e4, 1e9, 3.4e38])
@pytest.mark.parametrize("top", [1, 2])
def test_route_some_large_biases(hip, rng, kind, E, k, groups, keep, large, top):
    """experts, a pair in one group or a whole group moved far off by their bias; close scores"""
    z = np.round(16 * (1.5 * rng.standard_normal((60, E)))) / 16 + 2.0 ** -20 * rng.integers(0, 3, (60, E))
    bias = (0.05 * rng.standard_normal(E)).astype(np.float32)
    bias[[1, E // 2]] = large
    check(hip, kind, z, bias, k, groups, keep, top, least=0.2)
    bias[:E // 8] = large
    bias[E - 3] = -large
    check(hip, kind, z, bias, k, groups, keep, top, least=-1.0)


def time_us(hip, kind, z, bias, k, groups, keep):
    s, E = z.shape
    L = hip.lib()
    dz, db, di, dw = hip.DevBuf.from_array(z), hip.DevBuf.from_array(bias), hip.DevBuf(s * k * 4), hip.DevBuf(s * k * 4)
    cfg = hip.ApusHipRoute(KINDS[kind], k, groups, keep, 2, 1, 2.5)
    times = []
    for _ in range(7):
        hip.synchronize()
        L.apus_hip_timer_start()
        for _ in range(20):
            hip._check(L.apus_hip_route_dev(C.byref(cfg), dz.ptr, db.ptr, s, E, di.ptr, dw.ptr, None), "route")
        times.append(L.apus_hip_timer_stop() / 20 * 1e3)
    return sorted(times)[3]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("E,k,groups,keep", SHAPES[:5])
def test_route_a_large_bias_costs_little(hip, rng, kind, E, k, groups, keep):
    """an expert switched off by -1e9 or by -inf: about the same time (1.9 to 4.2 times
    where every token is ranked in 64 bits)"""
    z = (1.5 * rng.standard_normal((8192, E))).astype(np.float32)
    bias = (0.05 * rng.standard_normal(E)).astype(np.float32)
    off = bias.copy()
    bias[5], off[5] = -np.inf, -1e9
    a, b = (time_us(hip, kind, z, v, k, groups, keep) for v in (bias, off))
    assert b < 1.6 * a, (a, b)
