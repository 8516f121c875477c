"""Beams and long contexts over the KV caches, as timed cases.

Four operators, each called the way a serving loop calls the engine's C-ABI on
device buffers, beside a plain torch form of the same definition:

* window: attention of new tokens, a whole prompt or one token of each sequence,
  over caches that hold them already, causal, with a sliding window and a few
  first tokens that stay visible, or without a window;
* prefix: one query token of each sequence over a prefix that the sequences of a
  group share and over the sequence's own cache;
* select: the best continuations over the beams of a group and the vocabulary;
* reorder: the caches of a group's beams brought in line with that choice.

Caches are fp16, or e4m3 with one power-of-two scale for each sequence, head and
block of 32 tokens. Positions, lengths and parents are on the device.

`own` selects the engine's kernels; otherwise `run` computes the plain form.
Inputs are drawn on the GPU from the seed: queries and K / V rows ~N(0, 1),
logits ~N(0, 3^2), scores of beams a few units apart.
"""

import importlib
import math

import torch

own = False

KVB = 32  # tokens of a head that share a cache scale
U8, I32, I64 = torch.uint8, torch.int32, torch.int64
F8, F16, F32, F64 = torch.float8_e4m3fn, torch.float16, torch.float32, torch.float64

_ENG = None


def _engine():
    global _ENG
    if _ENG is None:
        _ENG = importlib.import_module("bare-metal-llm-engine_amd").Engine()
    return _ENG


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def _window(cache, batch, tokens, past, heads, kv_heads, dim, window, sinks, ragged):
    return {"op": "window", "cache": cache, "batch": batch, "tokens": tokens, "past": past,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks,
            "ragged": ragged}


def _prefix(cache, groups, beams, prefix, own_len, heads, kv_heads, dim):
    return {"op": "prefix", "cache": cache, "groups": groups, "beams": beams, "prefix": prefix,
            "own_len": own_len, "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _select(src, groups, beams, n_out, vocab, first):
    return {"op": "select", "src": src, "groups": groups, "beams": beams, "n_out": n_out,
            "vocab": vocab, "first": first}


def _reorder(cache, groups, beams, tokens, kv_heads, dim, in_place):
    return {"op": "reorder", "cache": cache, "groups": groups, "beams": beams, "tokens": tokens,
            "kv_heads": kv_heads, "dim": dim, "in_place": in_place}


def listed():
    return [
        # a 4096-token prompt through a layer with a sliding window, fp16 cache
        {"name": "prompt_4096_window", **_window("f16", 1, 4096, 0, 32, 8, 128, 1024, 4, False)},
        # eight prompts of unlike lengths, right-padded, on a small GQA model
        {"name": "prompts_777_ragged", **_window("q8", 8, 777, 0, 32, 4, 64, 256, 16, True)},
        # the last 2048 tokens of a prompt of 8192 that is written in pieces, all visible
        {"name": "prompt_piece_full", **_window("q8", 1, 2048, 6144, 32, 8, 128, 0, 0, False)},
        # sixteen sequences of unlike lengths decoded with a window and sinks
        {"name": "decode_16_window", **_window("q8", 16, 1, 8191, 32, 8, 128, 4096, 4, True)},
        # one token of one sequence, a short window: latency
        {"name": "decode_1_window", **_window("f16", 1, 1, 2047, 32, 32, 128, 512, 4, False)},
        # four beams over a prompt of 2000 tokens
        {"name": "prefix_4_beams", **_prefix("q8", 1, 4, 2000, 64, 32, 4, 64)},
        # thirty-two answers sampled from one long prompt
        {"name": "prefix_32_answers", **_prefix("f16", 1, 32, 8192, 500, 32, 8, 128)},
        # eight prompts with four beams each
        {"name": "prefix_8_groups", **_prefix("q8", 8, 4, 4096, 128, 32, 32, 128)},
        # the first step of a beam search over a 32000-word vocabulary
        {"name": "select_first", **_select("f32", 1, 4, 8, 32000, True)},
        # sixteen beam searches over a large vocabulary
        {"name": "select_16x4", **_select("f32", 16, 4, 8, 152064, False)},
        # the beams of one search, a few dozen tokens behind the prompt
        {"name": "reorder_4_beams", **_reorder("f16", 1, 4, 61, 8, 128, True)},
        # sixteen searches with 8-bit caches, into a second set of buffers
        {"name": "reorder_16x4", **_reorder("q8", 16, 4, 1000, 32, 128, False)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((32, 32, 128), (32, 8, 128), (64, 8, 128), (40, 40, 128), (12, 4, 64), (32, 4, 64),
         (8, 1, 64), (24, 2, 128))


def draw(rng):
    op = rng.choice(("window", "window", "prefix", "prefix", "select", "reorder"))
    cache = rng.choice(("f16", "q8"))
    heads, kv_heads, dim = rng.choice(HEADS)
    if op == "window":
        window = 0 if rng.random() < 0.3 else _log_int(rng, 1, 6000)
        sinks = rng.choice((0, 1, 4, 33, 130)) if window else 0
        if rng.random() < 0.5:  # a prompt, or a piece of one
            batch = _log_int(rng, 1, 12)
            tokens = _log_int(rng, 2, 4096)
            past = 0 if rng.random() < 0.5 else _log_int(rng, 1, 8192)
            most = 32 * 2048 * 8192 * 128
            while batch * heads * tokens * (tokens + past) * dim > most:
                batch, tokens, past = max(1, batch // 2), tokens - tokens // 4, past - past // 4
        else:
            batch, tokens, past = _log_int(rng, 1, 32), 1, _log_int(rng, 1, 30000) - 1
            past = min(past, 16 * 8192 * 8 * 128 // (batch * kv_heads * dim))
        return _window(cache, batch, tokens, past, heads, kv_heads, dim, window, sinks,
                       rng.random() < 0.6)
    if op == "prefix":
        groups, beams = _log_int(rng, 1, 12), _log_int(rng, 1, 48)
        prefix, own_len = _log_int(rng, 1, 16000), _log_int(rng, 1, 1000)
        groups = max(1, min(groups, 128 // beams))
        prefix = max(1, min(prefix, 32 * 4096 * 32 * 128 // (groups * beams * heads * dim)))
        return _prefix(cache, groups, beams, prefix, own_len, heads, kv_heads, dim)
    groups, beams = _log_int(rng, 1, 24), rng.randint(1, 10)
    if op == "select":
        vocab = _log_int(rng, 500, 152064)
        return _select("f32" if cache == "q8" else "f16", groups, beams,
                       beams * rng.choice((1, 2)), vocab, rng.random() < 0.2)
    tokens = _log_int(rng, 1, 2000)
    tokens = max(1, min(tokens, 64 * 1000 * 32 * 128 // (groups * beams * kv_heads * dim)))
    return _reorder(cache, groups, beams, tokens, kv_heads, dim, rng.random() < 0.5)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

class _Draws:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, shape, std, dtype):
        return (torch.randn(shape, generator=self.g, device="cuda", dtype=F32) * std).to(dtype)

    def uniform(self, shape):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=F32)

    def ints(self, lo, hi, shape):
        """Whole numbers of [lo, hi]."""
        return torch.randint(lo, hi + 1, shape, generator=self.g, device="cuda", dtype=I32)

    def cache(self, kind, n, heads, room, dim):
        """K or V of `n` sequences, head-major: {"c": fp16} or {"c": e4m3, "s": scales}."""
        x = self.normal((n, heads, room, dim), 1.0, F16)
        if kind == "f16":
            return {"c": x}
        x = x.view(n, heads, room // KVB, KVB, dim).to(F32)
        f, p = torch.frexp(x.abs().amax((-1, -2)))  # top = f 2^p; 448 = 0.875 2^9
        s = torch.ldexp(torch.ones_like(f), torch.where(f > 0.875, p - 8, p - 9))
        return {"c": (x / s[..., None, None]).to(F8).view(n, heads, room, dim), "s": s}


def _room(L):
    return -(-L // KVB) * KVB


def _inputs(case, seed):
    d = _Draws(seed)
    op = case["op"]
    if op == "window":
        B, S, past = case["batch"], case["tokens"], case["past"]
        room = _room(past + S)
        kv = [d.cache(case["cache"], B, case["kv_heads"], room, case["dim"]) for _ in range(2)]
        q = d.normal((B, S, case["heads"], case["dim"]), 1.0, F16)
        pos = torch.full((B,), past, device="cuda", dtype=I32)
        n = torch.full((B,), S, device="cuda", dtype=I32)
        if case["ragged"]:
            pos = d.ints(past // 4, past, (B,))
            n = d.ints((S + 1) // 2, S, (B,))
            pos[0], n[0] = past, S
        return {"q": q, "k": kv[0], "v": kv[1], "pos": pos, "n": n, "room": room}
    groups, beams = case["groups"], case["beams"]
    B = groups * beams
    if op == "prefix":
        G, D = case["kv_heads"], case["dim"]
        proom, room = _room(case["prefix"]), _room(case["own_len"])
        pk, pv = (d.cache(case["cache"], groups, G, proom, D) for _ in range(2))
        k, v = (d.cache(case["cache"], B, G, room, D) for _ in range(2))
        plen = d.ints(max(1, case["prefix"] * 3 // 4), case["prefix"], (groups,))
        plen[0] = case["prefix"]
        lens = d.ints(0, case["own_len"], (B,))
        return {"q": d.normal((B, case["heads"], D), 1.0, F16), "pk": pk, "pv": pv, "k": k, "v": v,
                "plen": plen, "lens": lens, "proom": proom, "room": room}
    if op == "select":
        ld = -(-case["vocab"] // 64) * 64  # a vocabulary padded by the last layer
        x = d.normal((B, ld), 3.0, F16 if case["src"] == "f16" else F32)
        scores = -10 - 4 * d.uniform((groups, beams))
        finished = (d.ints(0, 7, (groups, beams)) == 0).to(U8)
        if case["first"]:  # one live beam, nothing finished
            scores = torch.where(torch.arange(beams, device="cuda") == 0, torch.zeros_like(scores),
                                 torch.full_like(scores, -math.inf))
            finished = torch.zeros_like(finished)
        return {"x": x, "scores": scores, "finished": finished, "ld": ld}
    room = _room(case["tokens"] + 1)
    k, v = (d.cache(case["cache"], B, case["kv_heads"], room, case["dim"]) for _ in range(2))
    lens = torch.full((B,), case["tokens"], device="cuda", dtype=I32)
    parent = d.ints(0, beams - 1, (groups, beams))
    if case["in_place"]:  # beams that live on stay where they are, the others are replaced
        alive = torch.zeros((groups, beams), device="cuda", dtype=torch.bool)
        alive.scatter_(1, parent.to(I64), True)
        own_slot = torch.arange(beams, device="cuda", dtype=I32).expand(groups, beams)
        parent = torch.where(alive, own_slot, parent)
    return {"k": k, "v": v, "lens": lens, "parent": parent, "room": room}


def prepare(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    new = lambda shape, dtype: torch.zeros(shape, device="cuda", dtype=dtype)  # noqa: E731
    if op in ("window", "prefix"):
        t["out"] = torch.zeros_like(t["q"])
    elif op == "select":
        shape = (case["groups"], case["n_out"])
        t.update(out_scores=new(shape, F32), out_parent=new(shape, I32), out_token=new(shape, I32),
                 out_finished=new(shape, U8))
    elif case["in_place"]:
        t.update(k2=t["k"], v2=t["v"])
    else:
        t.update(k2={n: torch.zeros_like(x) for n, x in t["k"].items()},
                 v2={n: torch.zeros_like(x) for n, x in t["v"].items()})
    return {"case": case, "t": t}


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

EOS = 2


def run(state):
    return (_run_own if own else _run_plain)(state["case"], state["t"])


def _pointers(t, names):
    """Device pointers of K / V pairs, the scales behind the values: k, v[, ks, vs]."""
    kv = [t[n] for n in names]
    return [x["c"].data_ptr() for x in kv] + [x["s"].data_ptr() for x in kv if "s" in x]


def _run_own(case, t):
    eng, op = _engine(), case["op"]
    a = {k: v.data_ptr() for k, v in t.items() if isinstance(v, torch.Tensor)}
    if op == "window":
        eng.call("eng_attention_window_" + case["cache"], a["q"], *_pointers(t, ("k", "v")), a["out"],
                 a["pos"], a["n"], case["batch"], case["tokens"], case["heads"], case["kv_heads"],
                 case["dim"], case["window"], case["sinks"], case["past"] + case["tokens"],
                 t["room"], 1 / math.sqrt(case["dim"]), 0, None)
        return t["out"]
    groups, beams = case["groups"], case["beams"]
    if op == "prefix":
        eng.call("eng_attention_prefix_" + case["cache"], a["q"], *_pointers(t, ("pk", "pv")), a["plen"],
                 *_pointers(t, ("k", "v")), a["lens"], a["out"], groups, groups * beams,
                 case["heads"], case["kv_heads"], case["dim"], case["prefix"], t["proom"],
                 case["own_len"], t["room"], 1 / math.sqrt(case["dim"]), 0, None)
        return t["out"]
    if op == "select":
        eng.call("eng_beam_select_" + case["src"], a["x"], t["ld"], a["scores"], a["finished"],
                 a["out_scores"], a["out_parent"], a["out_token"], a["out_finished"], groups, beams,
                 case["n_out"], case["vocab"], EOS, None)
        return {n: t["out_" + n] for n in ("scores", "parent", "token", "finished")}
    eng.call("eng_kv_cache_reorder_" + case["cache"], *_pointers(t, ("k", "v")), *_pointers(t, ("k2", "v2")),
             a["parent"], a["lens"], groups, beams, case["kv_heads"], case["dim"], case["tokens"],
             t["room"], None)
    return {"k": t["k2"], "v": t["v2"]}


def _values(cache, dtype):
    """The values a cache stands for, [n, heads, room, dim]."""
    c = cache["c"].to(dtype)
    if "s" not in cache:
        return c
    n, heads, room, dim = c.shape
    return (c.view(n, heads, -1, KVB, dim) * cache["s"].to(dtype)[..., None, None]).view(c.shape)


def _softmax(s, live):
    s = torch.where(live, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _run_plain(case, t):
    op = case["op"]
    if op == "window":
        B, S, H, D = t["q"].shape
        G, L = case["kv_heads"], t["room"]
        q = t["q"].to(F32).view(B, S, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
        k, v = _values(t["k"], F32), _values(t["v"], F32)
        s = torch.matmul(q, k.transpose(2, 3)).reshape(B, G, H // G, S, L) / math.sqrt(D)
        j = torch.arange(L, device=q.device)
        p = (t["pos"].view(B, 1) + torch.arange(S, device=q.device)).view(B, 1, 1, S, 1)
        live = j <= p
        if case["window"]:
            live = live & ((j > p - case["window"]) | (j < case["sinks"]))
        o = torch.matmul(_softmax(s, live).reshape(B, G, -1, L), v).reshape(B, H, S, D).permute(0, 2, 1, 3)
        rows = torch.arange(S, device=q.device).view(1, S, 1, 1) < t["n"].view(B, 1, 1, 1)
        return torch.where(rows, o.to(F16), t["out"])  # rows behind a sequence stay as they were
    groups, beams = case["groups"], case["beams"]
    if op == "prefix":
        B, H, D = t["q"].shape
        G = case["kv_heads"]
        q = t["q"].to(F32).view(groups, beams, G, H // G, D).transpose(1, 2).reshape(groups, G, -1, D)
        pk, pv = _values(t["pk"], F32), _values(t["pv"], F32)
        k, v = _values(t["k"], F32), _values(t["v"], F32)
        P, L = t["proom"], t["room"]
        sp = torch.matmul(q, pk.transpose(2, 3)).reshape(groups, G, beams, H // G, P)
        sp = sp.transpose(1, 2).reshape(B, G, H // G, P)
        so = torch.matmul(t["q"].to(F32).view(B, G, H // G, D), k.transpose(2, 3))
        lp = torch.arange(P, device=q.device) < t["plen"].repeat_interleave(beams).view(B, 1, 1, 1)
        lo = torch.arange(L, device=q.device) < t["lens"].view(B, 1, 1, 1)
        live = torch.cat((lp, lo), -1).expand(B, G, H // G, P + L)
        w = _softmax(torch.cat((sp, so), -1) / math.sqrt(D), live)
        wp = w[..., :P].reshape(groups, beams, G, H // G, P).transpose(1, 2).reshape(groups, G, -1, P)
        op_ = torch.matmul(wp, pv).reshape(groups, G, beams, H // G, D).transpose(1, 2).reshape(B, G, H // G, D)
        return (op_ + torch.matmul(w[..., P:], v)).reshape(B, H, D).to(F16)
    if op == "select":
        V = case["vocab"]
        x = t["x"][:, :V].to(F64)  # neighbours in rank may be a few 1e-7 apart
        top = x.amax(-1, keepdim=True)
        s = x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
        s = t["scores"].to(F64).view(groups, beams, 1) + s.view(groups, beams, V)
        done = t["finished"].bool().unsqueeze(-1)
        eos = torch.arange(V, device=x.device) == EOS
        s = torch.where(done, torch.where(eos, t["scores"].to(F64).unsqueeze(-1), torch.full_like(s, -math.inf)), s)
        best, at = torch.sort(s.view(groups, -1), stable=True, dim=-1, descending=True)
        best, at = best[:, :case["n_out"]], at[:, :case["n_out"]]
        parent, token = torch.div(at, V, rounding_mode="floor"), at % V
        finished = t["finished"].gather(1, parent).bool() | (token == EOS)
        return {"scores": best.to(F32), "parent": parent.to(I32), "token": token.to(I32),
                "finished": finished.to(U8)}
    L, B = case["tokens"], groups * beams
    at = (torch.arange(groups, device="cuda").view(-1, 1) * beams + t["parent"].to(I64)).view(-1)
    got = {}
    for side in ("k", "v"):
        old, new = t[side], t[side + "2"]
        new["c"].view(U8)[:, :, :L] = old["c"].view(U8)[at, :, :L]
        if "s" in old:
            nb = -(-L // KVB)
            new["s"][:, :, :nb] = old["s"][at, :, :nb]
        got[side] = new
    return got


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * (2 if case["src"] == "f16" else 4), "flops": 4 * n}
    G, D = case["kv_heads"], case["dim"]
    per = 2 * D * G * (2 if case["cache"] == "f16" else 1 + 4 / (KVB * D))  # bytes of a token's K and V
    if op == "reorder":
        # a random choice takes 1 - (1 - 1 / beams)^beams of the beams; in place those stay
        b = case["beams"]
        taken = 1 - (1 - 1 / b) ** b
        n = case["groups"] * b * case["tokens"]
        moved = (1 - taken) * 2 if case["in_place"] else taken + 1
        return {"bytes": int(n * moved * per) + 4 * case["groups"] * b, "flops": 0}
    H = case["heads"]
    if op == "prefix":
        B = case["groups"] * case["beams"]
        shared, mine = case["groups"] * case["prefix"] * 0.875, B * case["own_len"] * 0.5
        return {"bytes": int((shared + mine) * per + 4 * B * H * D),
                "flops": int(4 * H * D * (shared * case["beams"] + mine))}
    S, W, sinks = case["tokens"], case["window"], case["sinks"]
    past, rows = case["past"], case["tokens"]
    if case["ragged"]:
        past, rows = past * 0.625, rows * 0.75 if S > 1 else 1
    first, last = past + 1, past + rows  # keys of the first and the last query
    pairs = rows * (first + last) / 2
    keys = last
    if W:
        def seen(n):
            return n if n <= W + sinks else W + sinks
        pairs = sum(seen(first + (i + 0.5) * rows / 64 - 0.5) for i in range(64)) * rows / 64
        keys = min(last, W + rows + sinks)
    return {"bytes": int(case["batch"] * (keys * per + 4 * rows * H * D)),
            "flops": int(4 * case["batch"] * H * D * pairs)}


# --------------------------------------------------------------------------
# results in 64 bits, from the definitions
# --------------------------------------------------------------------------

def _cache64(cache, b, heads=None):
    """K or V of sequence b in 64 bits, [heads, room, dim]."""
    c = cache["c"][b].to(F64)
    if "s" in cache:
        c = c * cache["s"][b].to(F64).repeat_interleave(KVB, 1).unsqueeze(-1)
    return c


def exact(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    dev = t["q"].device if "q" in t else "cuda"
    if op == "window":
        out = torch.zeros(t["q"].shape, device=dev, dtype=F64)
        W, sinks, group = case["window"], case["sinks"], case["heads"] // case["kv_heads"]
        for b, (p0, n) in enumerate(zip(t["pos"].tolist(), t["n"].tolist())):
            k, v = _cache64(t["k"], b), _cache64(t["v"], b)
            pos = torch.arange(p0, p0 + n, device=dev).view(-1, 1)
            key = torch.arange(p0 + n, device=dev).view(1, -1)
            hidden = key > pos
            if W:
                hidden |= (key < pos - W + 1) & (key >= sinks)
            for h in range(case["heads"]):
                s = t["q"][b, :n, h].to(F64) @ k[h // group, :p0 + n].t().contiguous() / math.sqrt(case["dim"])
                out[b, :n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[h // group, :p0 + n]
        return out
    groups, beams = case["groups"], case["beams"]
    if op == "prefix":
        B, H, D = t["q"].shape
        G = case["kv_heads"]
        out = torch.zeros((B, H, D), device=dev, dtype=F64)
        plen, lens = t["plen"].tolist(), t["lens"].tolist()
        for g in range(groups):
            pk, pv = (_cache64(t[n], g)[:, :plen[g]] for n in ("pk", "pv"))
            for b in range(g * beams, (g + 1) * beams):
                k = torch.cat((pk, _cache64(t["k"], b)[:, :lens[b]]), 1)
                v = torch.cat((pv, _cache64(t["v"], b)[:, :lens[b]]), 1)
                q = t["q"][b].to(F64).view(G, H // G, D)
                w = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D), -1)
                out[b] = torch.matmul(w, v).view(H, D)
        return out
    if op == "select":
        V, k = case["vocab"], case["n_out"]
        logp = torch.log_softmax(t["x"][:, :V].to(F64), -1).view(groups, beams, V)
        got = {n: [] for n in ("scores", "parent", "token", "finished")}
        for g in range(groups):
            names, values = [], []
            for b in range(beams):
                s = t["scores"][g, b].to(F64)
                if t["finished"][g, b]:
                    names.append(torch.tensor([b * V + EOS], device=dev))
                    values.append(s.view(1))
                else:
                    names.append(b * V + torch.arange(V, device=dev))
                    values.append(s + logp[g, b])
            names, values = torch.cat(names), torch.cat(values)
            if values.numel() < k:
                return None
            order = torch.sort(values, stable=True, dim=-1, descending=True)[1][:k]
            at = names[order]
            got["scores"].append(values[order])
            got["parent"].append(at // V)
            got["token"].append(at % V)
            got["finished"].append((t["finished"][g][at // V] != 0) | (at % V == EOS))
        return {n: torch.stack(v).to(F64 if n == "scores" else U8 if n == "finished" else I32)
                for n, v in got.items()}
    L, nb = case["tokens"], -(-case["tokens"] // KVB)
    got = {}
    for side in ("k", "v"):
        old = t[side]
        new = {n: (x.clone() if case["in_place"] else torch.zeros_like(x)) for n, x in old.items()}
        for g, row in enumerate(t["parent"].tolist()):
            for j, p in enumerate(row):
                new["c"][g * beams + j, :, :L] = old["c"][g * beams + p, :, :L]
                if "s" in old:
                    new["s"][g * beams + j, :, :nb] = old["s"][g * beams + p, :, :nb]
        got[side] = {n: x.to(F64) for n, x in new.items()}
    return got
