"""The 4-bit weights and the 8-bit cache together, as a decode loop uses them: one
transformer layer for three sequences, weights quantised on the device, prompts of
unlike lengths written into the cache, then single tokens. Each step's operators are
checked on the intermediates they were given (float64, each operator's own bound), and
the step is captured once and replayed with positions advancing on the device."""

from __future__ import annotations

import numpy as np
import pytest

import helpers
import narrow

pytestmark = pytest.mark.gpu
EPS = 1e-5
B, H, G, D, F, ROOM = 3, 8, 2, 64, 352, 96
E = H * D


class Layer:
    def __init__(self, gpu, seed):
        self.gpu = gpu
        rng = self.rng = np.random.default_rng(seed)
        self.W, self.dev = {}, {}
        for name, (n, k) in {"q": (E, E), "k": (G * D, E), "v": (G * D, E), "o": (E, E),
                             "gate": (F, E), "up": (F, E), "down": (E, F)}.items():
            w = gpu.upload((0.05 * rng.standard_normal((n, k))).astype(np.float32))
            nb = -(-k // 32)
            codes, scales = gpu.empty((n, nb * 16), np.uint8), gpu.empty((n, nb), np.uint8)
            gpu.call("eng_mx4_quantize_f32", w.ptr, codes.ptr, scales.ptr, n, k, None)
            gpu.sync()
            self.dev[name] = (codes, scales, n, k)
            self.W[name] = narrow.mx4_decode(codes.download(), scales.download(), k)
        self.g = (1 + 0.1 * rng.standard_normal(E)).astype(np.float32)
        self.dg = gpu.upload(self.g)
        nb = ROOM // 32
        self.kc, self.vc = gpu.empty((B, G, ROOM, D), np.uint8), gpu.empty((B, G, ROOM, D), np.uint8)
        self.ks, self.vs = gpu.empty((B, G, nb), np.float32), gpu.empty((B, G, nb), np.float32)
        for c in (self.kc, self.vc, self.ks, self.vs):
            c.fill_bytes(0xFF)  # NaN everywhere: nothing unwritten may reach a result
        self.pos, self.len = gpu.empty(B, np.int32), gpu.empty(B, np.int32)
        f, h = np.float32, np.uint16
        self.t = {"x": gpu.empty((B, E), f), "qf": gpu.empty((B, E), f), "kf": gpu.empty((B, G * D), f),
                  "vf": gpu.empty((B, G * D), f), "q": gpu.empty((B, H, D), h),
                  "k": gpu.empty((B, 1, G, D), h), "v": gpu.empty((B, 1, G, D), h),
                  "att": gpu.empty((B, H, D), h), "attf": gpu.empty((B, E), f),
                  "o": gpu.empty((B, E), f), "h": gpu.empty((B, E), f), "gate": gpu.empty((B, F), f),
                  "up": gpu.empty((B, F), f), "act": gpu.empty((B, F), f), "down": gpu.empty((B, E), f),
                  "y": gpu.empty((B, E), f)}

    def linear(self, name, x, y, stream, norm=False):
        codes, scales, n, k = self.dev[name]
        if norm:
            self.gpu.call("eng_rmsnorm_linear_mx4w_nk", x.ptr, self.dg.ptr, codes.ptr, scales.ptr,
                          y.ptr, B, n, k, EPS, stream)
        else:
            self.gpu.call("eng_linear_mx4w_nk", x.ptr, codes.ptr, scales.ptr, y.ptr, B, n, k, stream)

    def step(self, s):
        call, t = self.gpu.call, self.t
        for a, f in (("q", "qf"), ("k", "kf"), ("v", "vf")):
            self.linear(a, t["x"], t[f], s, norm=True)
            call("eng_cast_f32_to_f16", t[f].ptr, t[a].ptr, t[f].size, s)
        call("eng_kv_cache_write_q8", t["k"].ptr, t["v"].ptr, self.kc.ptr, self.vc.ptr, self.ks.ptr,
             self.vs.ptr, self.pos.ptr, None, B, 1, G, D, ROOM, s)
        call("eng_attention_decode_q8", t["q"].ptr, self.kc.ptr, self.vc.ptr, self.ks.ptr, self.vs.ptr,
             t["att"].ptr, self.len.ptr, B, H, G, D, ROOM, ROOM, 1 / np.sqrt(D), 2, s)
        call("eng_cast_f16_to_f32", t["att"].ptr, t["attf"].ptr, B * E, s)
        self.linear("o", t["attf"], t["o"], s)
        call("eng_vector_add_f32", t["x"].ptr, t["o"].ptr, t["h"].ptr, B * E, s)
        self.linear("gate", t["h"], t["gate"], s, norm=True)
        self.linear("up", t["h"], t["up"], s, norm=True)
        call("eng_swiglu_f32", t["gate"].ptr, t["up"].ptr, t["act"].ptr, B * F, s)
        self.linear("down", t["act"], t["down"], s)
        call("eng_vector_add_f32", t["h"].ptr, t["down"].ptr, t["y"].ptr, B * E, s)

    def prompt(self, lens):
        S = max(lens)
        kn, vn = ((self.rng.standard_normal((B, S, G, D))).astype(np.float16) for _ in range(2))
        dk, dv = self.gpu.upload(kn.view(np.uint16)), self.gpu.upload(vn.view(np.uint16))
        dp, dn = self.gpu.upload(np.zeros(B, np.int32)), self.gpu.upload(np.array(lens, np.int32))
        self.gpu.call("eng_kv_cache_write_q8", dk.ptr, dv.ptr, self.kc.ptr, self.vc.ptr, self.ks.ptr,
                      self.vs.ptr, dp.ptr, dn.ptr, B, S, G, D, ROOM, None)
        self.gpu.sync()

    def place(self, lens, x):
        self.pos.upload(np.array(lens, np.int32))
        self.len.upload(np.array(lens, np.int32) + 1)
        self.t["x"].upload(x)

    def state(self):
        return {k: v.download() for k, v in
                {**self.t, "kc": self.kc, "vc": self.vc, "ks": self.ks, "vs": self.vs}.items()}


def check_step(layer, before, after, lens):
    W, t = layer.W, after

    def lin(name, x, y, norm=False):
        y64, a = narrow.linear64(x, W[name], layer.g if norm else None, EPS if norm else None)
        helpers.assert_within(y, y64, narrow.linear_bound(y64, a, x.shape[1], norm), name)

    for a, f in (("q", "qf"), ("k", "kf"), ("v", "vf")):
        lin(a, t["x"], t[f], True)
    kc, vc, ks, vs = (before[n].copy() for n in ("kc", "vc", "ks", "vs"))
    narrow.kv_write(t["k"].view(np.float16).astype(np.float64), kc, ks, lens, None)
    narrow.kv_write(t["v"].view(np.float16).astype(np.float64), vc, vs, lens, None)
    assert narrow.same_codes(kc, t["kc"]) and narrow.same_codes(vc, t["vc"])
    assert np.array_equal(ks, t["ks"], equal_nan=True) and np.array_equal(vs, t["vs"], equal_nan=True)
    y, bound = narrow.attend64(t["q"].view(np.float16).astype(np.float64), kc, vc, ks, vs,
                               np.array(lens) + 1, 1 / np.sqrt(D))
    helpers.assert_within(t["att"].view(np.float16), y, bound, "attention")
    lin("o", t["attf"], t["o"])
    lin("gate", t["h"], t["gate"], True)
    lin("up", t["h"], t["up"], True)
    lin("down", t["act"], t["down"])
    assert np.array_equal(t["y"], t["h"] + t["down"]) and np.isfinite(t["y"]).all()


def test_a_decode_loop_step_by_step_and_replayed(gpu):
    rng = np.random.default_rng(21)
    lens = [40, 0, 63]
    xs = [rng.standard_normal((B, E)).astype(np.float32) for _ in range(6)]
    with gpu.stream() as s:
        eager = Layer(gpu, 8)
        eager.prompt(lens)
        states = []
        for i, x in enumerate(xs):
            now = [n + i for n in lens]
            eager.place(now, x)
            before = eager.state()
            eager.step(s.handle)
            s.sync()
            after = eager.state()
            check_step(eager, before, after, now)
            states.append(after)

        graphed = Layer(gpu, 8)
        graphed.prompt(lens)
        # the capture's eager forerunner runs on sequences that are all inactive
        graphed.place([-1, -1, -1], xs[0])
        graphed.step(s.handle)
        s.sync()
        graph = gpu.graph(s)
        with graph:
            graphed.step(s.handle)
        for i, x in enumerate(xs):
            graphed.place([n + i for n in lens], x)
            gpu.sync()
            graph.launch()
            # the program's own eager work on the same stream between the replays
            eager.step(s.handle)
            s.sync()
            got = graphed.state()
            for name in states[i]:
                assert np.array_equal(got[name].view(np.uint8), states[i][name].view(np.uint8)), \
                    f"token {i}: {name}"
        graph.destroy()
