"""The norm, routing and integer products together, as a layer uses them: the
residual stream is normed once, its fp32 rows go to the gate, its E4M3 codes to an
FP8 product and its integer codes to an integer product, and the routed experts
take the expert ids and weights; each step equal to the same step on its own.
The run is repeated on a lane and captured into a graph that is replayed between
eager calls."""
import ctypes as C

import numpy as np
import pytest

import rowops as R
from helpers import fp8_weights

pytestmark = pytest.mark.gpu

DIM, INTER, E, TOPK, EPS = 2048, 2048, 16, 6, 1e-6


class Layer:
    def __init__(self, hip, rng, s):
        self.hip, self.L, self.s = hip, hip.lib(), s
        L, up = self.L, hip.DevBuf.from_array
        err = C.create_string_buffer(256)
        self.store = L.apus_hip_store_create(1, E, DIM, INTER, err, 256)
        assert self.store, err.value
        hip._check(L.apus_hip_store_fill_random(self.store, 3), "fill")
        self.x_np = rng.standard_normal((s, DIM)).astype(np.float32)
        self.res_np = (2 * rng.standard_normal((s, DIM))).astype(np.float32)
        self.gamma_np = (1 + 0.2 * rng.standard_normal(DIM)).astype(np.float32)
        self.gate_np = (rng.standard_normal((E, DIM)) / 45).astype(np.float32)
        self.bias_np = (0.1 * rng.standard_normal(E)).astype(np.float32)
        self.w8_np, self.w8s_np = fp8_weights(rng, 512, DIM)
        self.wi_np = rng.integers(-127, 128, (320, DIM), dtype=np.int8)
        self.wis_np = (0.001 * (1 + rng.random(320))).astype(np.float32)
        (self.x, self.res, self.gamma, self.gate, self.bias, self.w8, self.w8s, self.wi, self.wis) = (
            up(v) for v in (self.x_np, self.res_np, self.gamma_np, self.gate_np, self.bias_np, self.w8_np, self.w8s_np,
                            self.wi_np, self.wis_np))
        n = s * DIM
        sizes = dict(r=4 * n, y=4 * n, c8=n, s8=n // 32, ci=n, si=4 * s, z=4 * s * E, idx=4 * s * TOPK, wgt=4 * s * TOPK,
                     o8=4 * s * 512, oi=4 * s * 320, ym=4 * n)
        self.b = {k: hip.DevBuf(v) for k, v in sizes.items()}
        self.ws = hip.DevBuf(L.apus_hip_moe_workspace(self.store, s, TOPK))
        self.cfg = hip.ApusHipRoute(hip.SCORE_SIGMOID, TOPK, 4, 2, 2, 1, 2.5)

    def run(self):
        hip, L, b, s = self.hip, self.L, self.b, self.s
        c = hip._check
        c(L.apus_hip_rmsnorm_dev(self.x.ptr, DIM, self.res.ptr, b["r"].ptr, self.gamma.ptr, s, DIM, EPS, hip.R_OUT,
                                 b["y"].ptr, b["c8"].ptr, b["s8"].ptr), "norm")
        c(L.apus_hip_rmsnorm_dev(b["r"].ptr, DIM, None, None, self.gamma.ptr, s, DIM, EPS, hip.Q_I8, None, b["ci"].ptr,
                                 b["si"].ptr), "norm i8")
        c(L.apus_hip_wlinear_dev(self.gate.ptr, b["y"].ptr, b["z"].ptr, s, DIM, E, 0), "gate")
        c(L.apus_hip_route_dev(C.byref(self.cfg), b["z"].ptr, self.bias.ptr, s, E, b["idx"].ptr, b["wgt"].ptr, None), "route")
        c(L.apus_hip_fp8_gemm_dev(self.w8.ptr, self.w8s.ptr, b["c8"].ptr, b["s8"].ptr, b["o8"].ptr, s, 512, DIM, 0), "fp8")
        c(L.apus_hip_i8_gemm_dev(self.wi.ptr, self.wis.ptr, b["ci"].ptr, b["si"].ptr, b["oi"].ptr, s, 320, DIM, 0), "i8")
        c(L.apus_hip_moe_routed_dev(self.store, 0, b["y"].ptr, b["idx"].ptr, b["wgt"].ptr, s, TOPK, 10.0, b["ym"].ptr,
                                    self.ws.ptr), "experts")

    def take(self):
        s = self.s
        shape = dict(r=(s, DIM), y=(s, DIM), s8=(s, DIM // 128), si=(s,), z=(s, E), wgt=(s, TOPK), o8=(s, 512), oi=(s, 320),
                     ym=(s, DIM))
        out = {k: self.b[k].to_array(np.float32, v) for k, v in shape.items()}
        out["c8"] = self.b["c8"].to_array(np.uint8, (s, DIM))
        out["ci"] = self.b["ci"].to_array(np.int8, (s, DIM))
        out["idx"] = self.b["idx"].to_array(np.int32, (s, TOPK))
        return out

    def wipe(self):
        self.hip.synchronize()
        for v in self.b.values():
            z = np.full(v.nbytes, 0xEE, np.uint8)
            self.hip._check(self.L.apus_hip_h2d(v.ptr, z.ctypes.data, v.nbytes), "wipe")

    def close(self):
        self.hip.synchronize()
        self.L.apus_hip_store_free(self.store)


@pytest.fixture(params=[1, 5, 40])
def layer(request, hip, rng):
    lay = Layer(hip, rng, request.param)
    yield lay
    lay.close()


def same(a, b):
    return all(np.array_equal(a[k], b[k]) for k in a)


def test_chain_against_the_formulas(layer, hip, oracle):
    layer.run()
    o = layer.take()
    assert np.array_equal(o["r"], layer.x_np + layer.res_np)
    truth = R.norm_truth(o["r"], layer.gamma_np, EPS)
    assert (np.abs(o["y"] - truth) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(truth)).all()
    c8, s8 = R.quant_e4m3(oracle, o["y"])
    ci, si = R.quant_i8(o["y"])
    assert np.array_equal(o["c8"], c8) and np.array_equal(o["s8"], s8)
    assert np.array_equal(o["ci"], ci) and np.array_equal(o["si"], si)
    idx, wgt, _, gap = R.route("sigmoid", o["z"], layer.bias_np, TOPK, 4, 2, 2, 1, 2.5)
    assert (gap > 2.0 ** -40).all() and np.array_equal(o["idx"], idx)
    assert (np.abs(o["wgt"] - wgt) <= (2.0 ** -24 + 2.0 ** -40) * wgt).all()
    assert np.array_equal(o["oi"], R.product(ci, si, layer.wi_np, layer.wis_np))
    # the FP8 product and the experts on codes, ids and weights computed apart
    up = hip.DevBuf.from_array
    L, s = layer.L, layer.s
    kc, ks, ki, kw, ky = up(c8), up(s8), up(idx), up(o["wgt"]), up(o["y"])
    o8, ym = hip.DevBuf(s * 512 * 4), hip.DevBuf(s * DIM * 4)
    hip._check(L.apus_hip_fp8_gemm_dev(layer.w8.ptr, layer.w8s.ptr, kc.ptr, ks.ptr, o8.ptr, s, 512, DIM, 0), "fp8")
    hip._check(L.apus_hip_moe_routed_dev(layer.store, 0, ky.ptr, ki.ptr, kw.ptr, s, TOPK, 10.0, ym.ptr,
                                         layer.ws.ptr), "experts")
    hip.synchronize()
    assert np.array_equal(o8.to_array(np.float32, (s, 512)), o["o8"])
    assert np.array_equal(ym.to_array(np.float32, (s, DIM)), o["ym"]) and np.abs(o["ym"]).max() > 0


def test_chain_on_a_lane(layer, hip):
    layer.run()
    want = layer.take()
    layer.wipe()
    hip._check(layer.L.apus_hip_lanes(2), "lanes")
    hip._check(layer.L.apus_hip_fork(), "fork")
    hip._check(layer.L.apus_hip_lane(1), "lane 1")
    try:
        layer.run()
    finally:
        hip._check(layer.L.apus_hip_join(), "join")
    assert same(layer.take(), want)


def test_chain_captured(layer, hip):
    """three replays with eager work and waits between them, the inputs changed before the last"""
    layer.run()
    want = layer.take()
    hip._check(layer.L.apus_hip_graph_begin(), "begin")
    layer.run()
    hip._check(layer.L.apus_hip_graph_end(), "end")
    for _ in range(3):
        layer.wipe()
        hip._check(layer.L.apus_hip_graph_replay(1), "replay")
        assert same(layer.take(), want)
        layer.wipe()
        layer.run()
        assert same(layer.take(), want)
    new = np.ascontiguousarray(layer.x_np[::-1] * np.float32(0.7))
    hip._check(layer.L.apus_hip_h2d(layer.x.ptr, new.ctypes.data, new.nbytes), "h2d")
    layer.wipe()
    hip._check(layer.L.apus_hip_graph_replay(2), "replay")
    got = layer.take()
    layer.wipe()
    layer.run()
    assert same(layer.take(), got) and not np.array_equal(got["y"], want["y"])


def test_products_on_two_lanes_at_once(hip, rng):
    """calls that overlap: the same weights, two batches, two lanes"""
    L = hip.lib()
    M, O, K = 33, 640, 1024
    w = rng.integers(-127, 128, (O, K), dtype=np.int8)
    sw = np.full(O, 0.01, np.float32)
    dw, dsw = hip.DevBuf.from_array(w), hip.DevBuf.from_array(sw)
    xs = [rng.standard_normal((M, K)).astype(np.float32) for _ in range(2)]
    dx = [hip.DevBuf.from_array(x) for x in xs]
    ws = [hip.DevBuf(L.apus_hip_i8_linear_workspace(M, K)) for _ in xs]
    out = [hip.DevBuf(M * O * 4) for _ in xs]
    hip._check(L.apus_hip_lanes(2), "lanes")
    for _ in range(5):
        hip._check(L.apus_hip_fork(), "fork")
        for i in range(2):
            hip._check(L.apus_hip_lane(i), "lane")
            hip._check(L.apus_hip_i8_linear_dev(dw.ptr, dsw.ptr, dx[i].ptr, out[i].ptr, M, K, O, 0, ws[i].ptr), "linear")
        hip._check(L.apus_hip_join(), "join")
    for i in range(2):
        q, s = R.quant_i8(R.round_bf16(xs[i]))
        assert np.array_equal(out[i].to_array(np.float32, (M, O)), R.product(q, s, w, sw))
