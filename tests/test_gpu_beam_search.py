"""The long-context operators together, as a beam search uses them: prompts of two groups
through one windowless attention layer into their own caches, then steps in which every
beam attends over its group's prompt and its own tokens, the logits choose the next beams
and the beams' caches follow. Each operator is checked on what it was given (float64, its
own bound); the whole search runs eagerly and as a replayed graph, bit for bit the same."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
import narrow
import test_gpu_beam as tb

pytestmark = pytest.mark.gpu
GROUPS, BEAMS, H, G, D, V, P, ROOM, EOS = 2, 3, 4, 2, 64, 97, 70, 32, 5
B, E = GROUPS * BEAMS, H * D


class Search:
    def __init__(self, gpu, kind, seed):
        self.gpu, self.kind = gpu, kind
        rng = self.rng = np.random.default_rng(seed)
        f, h, i = np.float32, np.uint16, np.int32
        up = lambda *s: gpu.upload((0.08 * rng.standard_normal(s)).astype(f))  # noqa: E731
        self.W = {n: up(E, m) for n, m in (("q", E), ("k", G * D), ("v", G * D), ("out", V))}
        self.embed = rng.standard_normal((V, E)).astype(f)
        el, nb = (h, 0) if kind == "f16" else (np.uint8, 1)

        def cache(n, room):
            c = [gpu.empty((n, G, room, D), el) for _ in range(2)]
            c += [gpu.empty((n, G, -(-room // 32)), f) for _ in range(2 * nb)]
            for a in c:
                a.fill_bytes(0xFF)  # NaN everywhere
            return c

        self.prefix, self.own = cache(GROUPS, P), cache(B, ROOM)
        self.plen = np.array([P, 41])
        self.t = {"x": gpu.empty((B, E), f), "qf": gpu.empty((B, E), f), "kf": gpu.empty((B, G * D), f),
                  "vf": gpu.empty((B, G * D), f), "q": gpu.empty((B, H, D), h), "k": gpu.empty((B, 1, G, D), h),
                  "v": gpu.empty((B, 1, G, D), h), "att": gpu.empty((B, H, D), h), "attf": gpu.empty((B, E), f),
                  "logits": gpu.empty((B, V), f), "pos": gpu.upload(np.zeros(B, i)), "len": gpu.upload(np.ones(B, i)),
                  "plen": gpu.upload(self.plen.astype(i)), "scores": gpu.empty((GROUPS, BEAMS), f),
                  "done": gpu.empty((GROUPS, BEAMS), np.uint8), "new_scores": gpu.empty((GROUPS, BEAMS), f),
                  "parent": gpu.empty((GROUPS, BEAMS), i), "token": gpu.empty((GROUPS, BEAMS), i),
                  "new_done": gpu.empty((GROUPS, BEAMS), np.uint8)}

    def append(self, k, v, cache, pos, n, batch, s_new, room, stream):
        """k, v [batch, s_new, G, D]; pos and n on the device (8 bits) or as numbers (fp16)."""
        if self.kind == "q8":
            self.gpu.call("eng_kv_cache_write_q8", k.ptr, v.ptr, *[c.ptr for c in cache], pos.ptr,
                          None if n is None else n.ptr, batch, s_new, G, D, room, stream)
            return
        for b in range(batch):
            row, at = b * s_new * G * D * 2, b * G * room * D * 2
            self.gpu.call("eng_kv_cache_write_f16", k.ptr + row, v.ptr + row, cache[0].ptr + at, cache[1].ptr + at,
                          s_new if n is None else int(n[b]), G, D, int(pos[b]), room, stream)

    def prompt(self):
        """Both prompts at once, right-padded: K / V into the prefix caches, and the rows' attention."""
        gpu, rng = self.gpu, self.rng
        q, k, v = (rng.standard_normal((GROUPS, P, n, D)).astype(np.float16) for n in (H, G, G))
        dq, dk, dv = (gpu.upload(a.view(np.uint16)) for a in (q, k, v))
        zero, n = np.zeros(GROUPS, np.int32), self.plen.astype(np.int32)
        dz, dn = gpu.upload(zero), gpu.upload(n)
        self.append(dk, dv, self.prefix, dz if self.kind == "q8" else zero, dn if self.kind == "q8" else n, GROUPS,
                    P, P, None)
        out = gpu.empty(q.shape, np.uint16)
        out.fill_bytes(0)
        for window, sinks in ((0, 0), (24, 3)):
            gpu.call("eng_attention_window_" + self.kind, dq.ptr, *[c.ptr for c in self.prefix], out.ptr, dz.ptr,
                     dn.ptr, GROUPS, P, H, G, D, window, sinks, P, P, 1 / np.sqrt(D), 0, None)
            gpu.sync()
            want = lc.window64(q.astype(np.float64), self.view(self.prefix), zero, n, window, sinks, P,
                               float(np.float32(1 / np.sqrt(D))))
            lc.check(out.download().view(np.float16), want, f"prompt, window {window}")

    def view(self, cache):
        """What a cache on the device stands for, as the float64 statements take it."""
        host = [c.download() for c in cache]

        class View:
            pass

        view = View()
        if self.kind == "f16":
            view.values = [a.view(np.float16).astype(np.float64) for a in host]
            view.vmax = np.nanmax(np.abs(view.values[1]), (2, 3), initial=0.0, where=~np.isnan(view.values[1]))
        else:
            view.values = [narrow.kv_values(c, s) for c, s in zip(host[:2], host[2:])]
            view.vmax = 448 * np.nanmax(np.where(np.isnan(host[3]), 0, host[3]), 2)
        return view

    def place(self, tokens, scores, done, step):
        t = self.t
        t["x"].upload(self.embed[tokens.reshape(-1)])
        t["scores"].upload(scores.astype(np.float32))
        t["done"].upload(done.astype(np.uint8))
        t["pos"].upload(np.full(B, step, np.int32))
        t["len"].upload(np.full(B, step + 1, np.int32))

    def step(self, s, at):
        call, t = self.gpu.call, self.t
        for a, f in (("q", "qf"), ("k", "kf"), ("v", "vf")):
            call("eng_matmul_f32", t["x"].ptr, self.W[a].ptr, t[f].ptr, B, self.W[a].shape[1], E, s)
            call("eng_cast_f32_to_f16", t[f].ptr, t[a].ptr, t[f].size, s)
        self.append(t["k"], t["v"], self.own, t["pos"] if self.kind == "q8" else [at] * B, None, B, 1, ROOM, s)
        call("eng_attention_prefix_" + self.kind, t["q"].ptr, *[c.ptr for c in self.prefix], t["plen"].ptr,
             *[c.ptr for c in self.own], t["len"].ptr, t["att"].ptr, GROUPS, B, H, G, D, P, P, ROOM, ROOM,
             1 / np.sqrt(D), 0, s)
        call("eng_cast_f16_to_f32", t["att"].ptr, t["attf"].ptr, B * E, s)
        call("eng_matmul_f32", t["attf"].ptr, self.W["out"].ptr, t["logits"].ptr, B, V, E, s)
        call("eng_beam_select_f32", t["logits"].ptr, V, t["scores"].ptr, t["done"].ptr, t["new_scores"].ptr,
             t["parent"].ptr, t["token"].ptr, t["new_done"].ptr, GROUPS, BEAMS, BEAMS, V, EOS, s)
        own = [c.ptr for c in self.own]
        call("eng_kv_cache_reorder_" + self.kind, *own, *own, t["parent"].ptr, t["len"].ptr, GROUPS, BEAMS, G, D,
             ROOM, ROOM, s)

    def run(self, steps, step, check=False):
        """The beams' tokens and scores after `steps` steps, each run by step(search, i)."""
        tokens = np.zeros((GROUPS, BEAMS), np.int32)
        scores = np.full((GROUPS, BEAMS), -np.inf)
        scores[:, 0] = 0
        done = np.zeros((GROUPS, BEAMS), bool)
        words = np.zeros((GROUPS, BEAMS, 0), np.int32)
        for i in range(steps):
            self.place(tokens, scores, done, i)
            before = [c.download() for c in self.own]
            step(self, i)
            t = {k: v.download() for k, v in self.t.items()}
            if check:
                self.check(before, t, i)
            parent = t["parent"]
            words = np.concatenate((np.take_along_axis(words, parent[..., None], 1), t["token"][..., None]), 2)
            tokens, scores, done = t["token"], t["new_scores"], t["new_done"]
        return words, scores

    def check(self, before, t, i):
        f16 = lambda a: a.view(np.float16).astype(np.float64)  # noqa: E731
        if self.kind == "q8":
            (k, v, ks, vs), at = before, np.full(B, i)
            narrow.kv_write(f16(t["k"]), k, ks, at, None)
            narrow.kv_write(f16(t["v"]), v, vs, at, None)
            own = [k, v, ks, vs]
        else:
            own = [a.copy() for a in before]
            own[0][:, :, i], own[1][:, :, i] = t["k"][:, 0], t["v"][:, 0]
        device = [self.gpu.upload(a) for a in own]
        want = lc.prefix64(f16(t["q"]), self.view(self.prefix), self.plen, self.view(device), [i + 1] * B,
                           float(np.float32(1 / np.sqrt(D))))
        lc.check(t["att"].view(np.float16), want, f"step {i}: attention")
        got = [t[n] for n in ("new_scores", "parent", "token", "new_done")]
        tb.check(got, t["logits"].reshape(GROUPS, BEAMS, V), t["scores"], t["done"], BEAMS, EOS)
        for n, (a, d) in enumerate(zip(own, self.own)):
            m = i + 1 if n < 2 else -(-(i + 1) // 32)
            moved = a.reshape(GROUPS, BEAMS, *a.shape[1:])[np.arange(GROUPS)[:, None], t["parent"]]
            assert np.array_equal(d.download()[:, :, :m], moved.reshape(a.shape)[:, :, :m]), f"step {i}: cache {n}"


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_a_beam_search_step_by_step(gpu, kind):
    search = Search(gpu, kind, 3)
    search.prompt()

    def eager(s, i):
        s.step(None, i)
        gpu.sync()

    words, scores = search.run(8, eager, check=True)
    assert np.isfinite(scores).all() and (np.diff(scores, axis=1) <= 0).all()
    assert len({tuple(w) for w in words.reshape(-1, 8)}) > GROUPS


def test_the_same_search_replayed(gpu):
    """With 8-bit caches positions are on the device, so one captured step serves all."""
    def eager(s, i):
        s.step(None, i)
        gpu.sync()

    one = Search(gpu, "q8", 4)
    one.prompt()
    want = one.run(10, eager)
    with gpu.stream() as stream:
        two = Search(gpu, "q8", 4)
        two.prompt()
        two.t["pos"].upload(np.full(B, -1, np.int32))  # the capture's forerunner leaves the caches alone
        two.t["len"].upload(np.zeros(B, np.int32))
        for n in ("x", "scores", "done"):
            two.t[n].fill_bytes(0)
        gpu.sync()
        two.step(stream.handle, 0)
        stream.sync()
        graph = gpu.graph(stream)
        with graph:
            two.step(stream.handle, 0)

        def replay(s, i):
            gpu.sync()
            graph.launch()
            one.step(stream.handle, 0)  # eager work of another search between the replays
            stream.sync()

        got = two.run(10, replay)
        graph.destroy()
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
