"""Calls that apus_hip_rmsnorm_dev, _route_dev, _i8_quant_dev, _i8_gemm_dev and
_i8_linear_dev refuse: before any device work, so these run without a GPU (no
pointer here is read)."""
import ctypes as C

import pytest

import apus_hip as H

A = 0x10000000
P = [A + i * 0x1000000 for i in range(12)]      # far apart, 16-byte aligned


def refused(rc, word):
    assert rc != 0
    assert word in H.lib().apus_hip_last_error().decode(), H.lib().apus_hip_last_error()


def norm(**kw):
    a = dict(x=P[0], ldx=256, res=P[1], res_out=P[2], gamma=P[3], M=4, K=256, eps=1e-6, flags=0, y=P[4], codes=P[5],
             scales=P[6])
    a.update(kw)
    return H.lib().apus_hip_rmsnorm_dev(*a.values())


def test_norm_refusals():
    for kw in (dict(flags=1), dict(flags=64), dict(flags=-1)):
        refused(norm(**kw), "flags")
    for kw in (dict(M=-1), dict(K=0), dict(K=-128), dict(ldx=255), dict(K=200, ldx=200), dict(K=0x7fffffff, ldx=0x7fffffff),
               dict(M=0x7fffffff)):
        refused(norm(**kw), "shape")
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        refused(norm(eps=eps), "eps")
    for kw in (dict(x=None), dict(gamma=None), dict(scales=None), dict(codes=None), dict(res=None),
               dict(res=None, res_out=None, y=None, codes=None, scales=None)):
        refused(norm(**kw), "needed")
    for kw in (dict(x=P[0] + 2), dict(res=P[1] + 1), dict(res_out=P[2] + 2), dict(gamma=P[3] + 2), dict(y=P[4] + 2),
               dict(scales=P[6] + 1), dict(x=P[0] + 1, flags=H.X_BF16), dict(y=P[4] + 1, flags=H.Y_BF16),
               dict(gamma=P[3] + 1, flags=H.W_BF16)):
        refused(norm(**kw), "misaligned")


def test_norm_overlaps():
    refused(norm(res_out=P[0], ldx=300), "overlaps an input")            # over x whose rows lie apart
    refused(norm(y=P[0], flags=H.Y_BF16), "overlaps an input")           # another type
    refused(norm(y=P[1], flags=H.X_BF16), "overlaps an input")
    refused(norm(res_out=P[0] + 4), "overlaps an input")
    refused(norm(res_out=P[1] + 1024), "overlaps an input")
    refused(norm(y=P[3]), "overlaps an input")
    refused(norm(codes=P[0]), "overlaps an input")
    refused(norm(scales=P[1] + 4 * 256 * 4 - 4), "overlaps an input")
    refused(norm(y=P[2]), "two outputs")
    refused(norm(codes=P[4] + 4 * 256 * 4 - 1), "two outputs")
    refused(norm(scales=P[5] + 4 * 256 - 4), "two outputs")
    refused(norm(res_out=P[0], y=P[0]), "two outputs")


def route(change=None, **kw):
    c = dict(score=1, topk=8, n_group=8, topk_group=4, group_top=2, renorm=1, route_scale=2.5)
    c.update(change or {})
    a = dict(cfg=C.byref(H.ApusHipRoute(*c.values())), logits=P[0], bias=P[1], s=4, E=256, idx=P[2], wgt=P[3], scores=P[4])
    a.update(kw)
    return H.lib().apus_hip_route_dev(*a.values())


def test_route_refusals():
    refused(route(None, cfg=None), "bad score")
    for c in (dict(score=-1), dict(score=3), dict(renorm=2), dict(renorm=-1), dict(route_scale=float("inf")),
              dict(route_scale=float("nan"))):
        refused(route(c), "bad score")
    for kw in (dict(s=-1), dict(E=0), dict(E=1025), dict(s=0x7fffffff)):
        refused(route(None, **kw), "shape")
    for c in (dict(topk=0), dict(topk=17), dict(topk=-1)):
        refused(route(c), "shape")
    for c in (dict(n_group=0), dict(n_group=7), dict(n_group=128), dict(topk_group=0), dict(topk_group=9), dict(group_top=0),
              dict(group_top=3), dict(n_group=64, topk_group=1)):
        refused(route(c), "groups")
    refused(route(dict(n_group=1, topk_group=1), E=4), "groups")
    for kw in (dict(logits=None), dict(idx=None), dict(wgt=None), dict(logits=P[0] + 2), dict(bias=P[1] + 1),
               dict(idx=P[2] + 2), dict(wgt=P[3] + 3), dict(scores=P[4] + 2)):
        refused(route(None, **kw), "misaligned")
    for kw in (dict(scores=P[0]), dict(idx=P[1]), dict(wgt=P[0] + 4 * 256 * 4 - 4)):
        refused(route(None, **kw), "overlaps an input")
    refused(route(None, wgt=P[2]), "two outputs")


def test_i8_refusals():
    L = H.lib()

    def quant(x=P[0], M=4, K=256, flags=0, codes=P[1], scales=P[2]):
        return L.apus_hip_i8_quant_dev(x, M, K, flags, codes, scales)

    refused(quant(flags=16), "flags")
    for kw in (dict(M=-1), dict(K=0), dict(M=0x7fffffff), dict(K=0x7fffffff)):
        refused(quant(**kw), "shape")
    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(x=P[0] + 2), dict(x=P[0] + 1, flags=H.X_BF16),
               dict(scales=P[2] + 2)):
        refused(quant(**kw), "misaligned")
    refused(quant(codes=P[0] + 16), "overlaps an input")
    refused(quant(scales=P[1] + 1020), "two outputs")

    def gemm(w=P[0], ws=P[1], a=P[2], sa=P[3], out=P[4], M=4, O=64, K=256, flags=0):
        return L.apus_hip_i8_gemm_dev(w, ws, a, sa, out, M, O, K, flags)

    def linear(w=P[0], ws=P[1], x=P[2], out=P[4], M=4, K=256, O=64, flags=0, space=P[5]):
        return L.apus_hip_i8_linear_dev(w, ws, x, out, M, K, O, flags, space)

    for f in (gemm, linear):
        for kw in (dict(M=-1), dict(O=0), dict(K=0), dict(K=-4), dict(K=6), dict(K=131072), dict(M=0x7fffffff), dict(O=0x7fffffff)):
            refused(f(**kw), "shape")
        refused(f(flags=1), "flags")
        refused(f(flags=32), "flags")
        for kw in (dict(w=None), dict(ws=None), dict(out=None), dict(w=P[0] + 2), dict(ws=P[1] + 2), dict(out=P[4] + 2),
                   dict(out=P[4] + 1, flags=H.Y_BF16)):
            refused(f(**kw), "misaligned")
        refused(f(out=P[0]), "overlaps an input")
    refused(gemm(flags=8), "flags")
    for kw in (dict(a=None), dict(sa=None), dict(a=P[2] + 2), dict(sa=P[3] + 2)):
        refused(gemm(**kw), "misaligned")
    refused(gemm(out=P[3] + 12), "overlaps an input")
    for kw in (dict(x=None), dict(x=P[2] + 2), dict(x=P[2] + 1, flags=H.X_BF16)):
        refused(linear(**kw), "misaligned")
    for kw in (dict(space=None), dict(space=P[5] + 8)):
        refused(linear(**kw), "workspace")
    refused(linear(space=P[2]), "overlaps an input")
    refused(linear(space=P[4]), "two outputs")


def test_nothing_to_do():
    """no rows: done, without a device"""
    assert norm(M=0) == 0
    assert route(None, s=0) == 0
    L = H.lib()
    assert L.apus_hip_i8_quant_dev(P[0], 0, 256, 0, P[1], P[2]) == 0
    assert L.apus_hip_i8_gemm_dev(P[0], P[1], P[2], P[3], P[4], 0, 64, 256, 0) == 0
    assert L.apus_hip_i8_linear_dev(P[0], P[1], P[2], P[4], 0, 256, 64, 0, P[5]) == 0


@pytest.mark.parametrize("M,K,n", [(0, 256, 0), (-1, 256, 0), (4, 0, 0), (1, 4, 512), (3, 100, 768), (100000, 100000, 10000400128)])
def test_i8_linear_workspace(M, K, n):
    assert H.lib().apus_hip_i8_linear_workspace(M, K) == n
