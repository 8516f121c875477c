"""Decode with narrow storage: 4-bit weights and an 8-bit KV cache, as timed cases.

Four operators, each called the way a serving loop calls the engine's C-ABI on
device buffers, beside a plain torch form of the same definition:

* pack: weights to microscaled 4-bit floating point (E2M1 values, one E8M0
  scale byte for 32 values along a row) and back to the values they stand for;
* linear: y = x . W^T with such weights, fp32 x and y, with the RMSNorm of the
  rows folded in or without it, from one decoded token to a long prompt;
* write: new K / V rows into an e4m3 cache with one power-of-two scale for
  each sequence, head and block of 32 tokens, at a position of each sequence's
  own;
* attention: one query token of each sequence over such a cache, lengths on
  the device.

`own` selects the engine's kernels; otherwise `run` computes the plain form.
Inputs are drawn on the GPU from the seed: weights ~N(0, 0.02^2), activations
and K / V rows ~N(0, 1), RMSNorm gains 1 + N(0, 0.1^2).
"""

import importlib
import math

import torch

own = False

EPS = 1e-5
MXB = 32  # values along a row that share a scale byte
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

def _pack(rows, cols, src):
    return {"op": "pack", "rows": rows, "cols": cols, "src": src}


def _linear(M, N, K, norm):
    return {"op": "linear", "M": M, "N": N, "K": K, "norm": norm}


def _write(batch, tokens, kv_heads, dim, room, ragged):
    return {"op": "write", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "dim": dim,
            "room": room, "ragged": ragged}


def _attention(batch, L, heads, kv_heads, dim, ragged):
    return {"op": "attention", "batch": batch, "L": L, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "ragged": ragged}


def listed():
    return [
        # a loader packing a gate matrix of the 7B stack from its fp16 file
        {"name": "pack_gate_f16", **_pack(11008, 4096, "f16")},
        # a small fp32 matrix, rows that end inside a block of 32
        {"name": "pack_ragged_f32", **_pack(509, 1023, "f32")},
        # one decoded token through an attention output projection
        {"name": "decode_out_proj", **_linear(1, 4096, 4096, False)},
        # one decoded token through RMSNorm and the FFN's gate
        {"name": "decode_gate", **_linear(1, 11008, 4096, True)},
        # sixteen sequences decoded together: the FFN's gate
        {"name": "batch_16_gate", **_linear(16, 11008, 4096, True)},
        # a short ragged batch through a layer no side of which suits a tile
        {"name": "batch_ragged", **_linear(37, 2051, 1023, True)},
        # a 512-token prompt through the gate
        {"name": "prompt_512_gate", **_linear(512, 11008, 4096, True)},
        # one token of each of 32 sequences into their caches, MHA
        {"name": "append_32", **_write(32, 1, 32, 128, 2048, True)},
        # four prompts of up to 1000 tokens, right-padded, into their caches
        {"name": "prompts_1000", **_write(4, 1000, 8, 128, 2048, True)},
        # decode attention of a small GQA model in the middle of its context
        {"name": "attention_2048_gqa", **_attention(1, 2048, 32, 4, 64, False)},
        # one long MHA sequence
        {"name": "attention_8192_mha", **_attention(1, 8192, 32, 32, 128, False)},
        # sixteen sequences of unlike lengths (some without a token) on GQA
        {"name": "attention_16_ragged", **_attention(16, 8192, 32, 8, 128, True)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, unit):
    """A layer width: mostly a multiple of `unit`, one in four any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(unit, n // unit * unit)


HEADS = ((32, 32, 128), (32, 8, 128), (64, 8, 128), (40, 40, 128), (12, 4, 64), (32, 4, 64),
         (8, 1, 64), (24, 2, 128))


def draw(rng):
    op = rng.choice(("pack", "linear", "linear", "write", "attention", "attention"))
    if op == "pack":
        cols = _width(rng, 33, 11008, 64)
        rows = min(_log_int(rng, 1, 11008), 11008 * 4096 // cols)
        return _pack(max(1, rows), cols, rng.choice(("f16", "f32")))
    if op == "linear":
        N, K = _width(rng, 200, 14336, 64), _width(rng, 100, 11008, 64)
        M = _log_int(rng, 1, 1024)
        return _linear(max(1, min(M, 512 * 11008 * 4096 // (N * K))), N, K, rng.random() < 0.5)
    heads, kv_heads, dim = rng.choice(HEADS)
    batch = _log_int(rng, 1, 48)
    if op == "write":
        tokens = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1500)
        tokens = max(1, min(tokens, 4096 * 1024 // (batch * kv_heads * dim)))
        return _write(batch, tokens, kv_heads, dim, tokens + _log_int(rng, 1, 600), rng.random() < 0.7)
    L = _log_int(rng, 1, 40000)
    L = max(1, min(L, 16 * 8192 * 8 * 128 // (batch * kv_heads * dim)))
    return _attention(batch, L, heads, kv_heads, dim, batch > 1 and rng.random() < 0.7)


# --------------------------------------------------------------------------
# the formats, in elementary operations
# --------------------------------------------------------------------------

def _ldexp(x, e):
    """x 2^e, the power taken in two halves that 32 bits hold."""
    h = torch.div(e, 2, rounding_mode="floor")
    return torch.ldexp(torch.ldexp(x, h), e - h)


def _blocks_of(x, size):
    """x [rows, cols] as [rows, blocks, size], the last block filled with zeros."""
    rows, cols = x.shape
    nb = -(-cols // size)
    p = torch.zeros((rows, nb * size), device=x.device, dtype=x.dtype)
    p[:, :cols] = x
    return p.view(rows, nb, size)


def _mx4_encode(x):
    """x [rows, cols] fp32 -> codes [rows, 16 blocks], scale bytes [rows, blocks].

    2^e: floor(log2 of the block's largest magnitude) - 2, at least 2^-127;
    values over 6 2^e become 6, ties go to the even code."""
    x = _blocks_of(x, MXB)
    a = x.abs()
    top = a.amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    # frexp: top = f 2^p with f in [0.5, 1)
    p = torch.frexp(torch.where(bad, torch.ones_like(top), top))[1]
    e = torch.where(top == 0, torch.full_like(p, -127), p - 3).clamp(-127, 127)
    m = _ldexp(a, -e.unsqueeze(-1).expand(a.shape))
    code = ((m > 0.25).to(U8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5)
            + (m > 5.0))
    code = code + 8 * torch.signbit(x).to(U8)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).to(U8)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(U8)
    return codes.reshape(codes.shape[0], -1).contiguous(), scales.contiguous()


def _mx4_values(codes, scales, cols):
    """The fp32 values that codes and scales stand for, [rows, cols]."""
    rows = codes.shape[0]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0,
                         -3.0, -4.0, -6.0], device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1, MXB)
    v = _ldexp(grid[c.to(I64)], (scales.to(I32) - 127).unsqueeze(-1).expand(c.shape))
    v = torch.where((scales == 255).unsqueeze(-1), torch.full_like(v, float("nan")), v)
    return v.reshape(rows, -1)[:, :cols]


def _kv_scale(top):
    """The least 2^e, e in [-15, 8], with top <= 448 2^e (448 = 0.875 2^9)."""
    f, p = torch.frexp(top)
    e = torch.where(f > 0.875, p - 8, p - 9)
    e = torch.where(top == 0, torch.full_like(e, -15), e).clamp(-15, 8)
    return torch.ldexp(torch.ones_like(top), e)


def _kv_encode(x):
    """K or V rows [batch, heads, tokens, dim] fp16 -> e4m3 and scales, tokens a multiple of 32."""
    B, G, L, D = x.shape
    x = x.view(B, G, L // KVB, KVB, D).to(F32)
    s = _kv_scale(x.abs().amax((-1, -2)))
    return (x / s[..., None, None]).to(F8).view(B, G, L, D), s


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

    def gain(self, n):
        return 1 + 0.1 * torch.randn(n, generator=self.g, device="cuda", dtype=F32)

    def ints(self, lo, hi, n):
        """n whole numbers of [lo, hi]."""
        return torch.randint(lo, hi + 1, (n,), generator=self.g, device="cuda", dtype=I32)


def _room(L):
    return -(-L // KVB) * KVB


def _inputs(case, seed):
    d = _Draws(seed)
    op = case["op"]
    if op == "pack":
        return {"W": d.normal((case["rows"], case["cols"]), 0.02, F16 if case["src"] == "f16" else F32)}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        codes, scales = _mx4_encode(d.normal((N, K), 0.02, F16).to(F32))
        return {"x": d.normal((M, K), 1.0, F32), "g": d.gain(K), "codes": codes, "scales": scales}
    B, G, D = case["batch"], case["kv_heads"], case["dim"]
    if op == "write":
        S, room = case["tokens"], _room(case["room"])
        # a cache in use, and new rows a quarter of which are larger than what it holds
        kc, ks = _kv_encode(d.normal((B, G, room, D), 1.0, F16))
        vc, vs = _kv_encode(d.normal((B, G, room, D), 1.0, F16))
        grown = 1 + 2 * (d.ints(0, 3, B) == 0).to(F32).view(B, 1, 1, 1)
        kn = (d.normal((B, S, G, D), 1.0, F32) * grown).to(F16)
        vn = (d.normal((B, S, G, D), 1.0, F32) * grown).to(F16)
        pos = d.ints(0, room - S, B) if case["ragged"] else torch.full((B,), room - S, device="cuda", dtype=I32)
        n = d.ints((S + 1) // 2, S, B) if case["ragged"] else torch.full((B,), S, device="cuda", dtype=I32)
        return {"kn": kn, "vn": vn, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "pos": pos, "n": n}
    L, room = case["L"], _room(case["L"])
    kc, ks = _kv_encode(d.normal((B, G, room, D), 1.0, F16))
    vc, vs = _kv_encode(d.normal((B, G, room, D), 1.0, F16))
    lens = torch.full((B,), L, device="cuda", dtype=I32)
    if case["ragged"]:
        lens = d.ints(0, L, B)
        lens[0] = L
        lens[B // 2] = 0
    return {"q": d.normal((B, case["heads"], D), 1.0, F16), "kc": kc, "vc": vc, "ks": ks, "vs": vs,
            "lens": lens}


def prepare(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    new = lambda shape, dtype=F32: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    if op == "pack":
        rows, cols = case["rows"], case["cols"]
        nb = -(-cols // MXB)
        t.update(codes=new((rows, 16 * nb), U8), scales=new((rows, nb), U8),
                 out=new((rows, cols), t["W"].dtype))
    elif op == "linear":
        t["out"] = new((case["M"], case["N"]))
    elif op == "attention":
        t["out"] = new(t["q"].shape, F16)
    return {"case": case, "t": t, "engine": _engine()}


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    case, t = state["case"], state["t"]
    return (_run_own if own else _run_plain)(case, t, state["engine"])


def _run_own(case, t, eng):
    op = case["op"]
    a = {k: v.data_ptr() for k, v in t.items()}
    if op == "pack":
        rows, cols, src = case["rows"], case["cols"], case["src"]
        eng.call("eng_mx4_quantize_" + src, a["W"], a["codes"], a["scales"], rows, cols, None)
        eng.call("eng_mx4_dequantize_" + src, a["codes"], a["scales"], a["out"], rows, cols, None)
        return {"values": t["out"], "scales": t["scales"]}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        if case["norm"]:
            eng.call("eng_rmsnorm_linear_mx4w_nk", a["x"], a["g"], a["codes"], a["scales"],
                     a["out"], M, N, K, EPS, None)
        else:
            eng.call("eng_linear_mx4w_nk", a["x"], a["codes"], a["scales"], a["out"], M, N, K, None)
        return t["out"]
    B, G, D = case["batch"], case["kv_heads"], case["dim"]
    room = t["kc"].shape[2]
    if op == "write":
        eng.call("eng_kv_cache_write_q8", a["kn"], a["vn"], a["kc"], a["vc"], a["ks"], a["vs"],
                 a["pos"], a["n"], B, case["tokens"], G, D, room, None)
        return {"k": t["kc"], "v": t["vc"], "k_scale": t["ks"], "v_scale": t["vs"]}
    eng.call("eng_attention_decode_q8", a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["out"],
             a["lens"], B, case["heads"], G, D, case["L"], room, 1 / math.sqrt(D), 0, None)
    return t["out"]


def _run_plain(case, t, eng):
    op = case["op"]
    if op == "pack":
        codes, scales = _mx4_encode(t["W"].to(F32))
        return {"values": _mx4_values(codes, scales, case["cols"]).to(t["W"].dtype), "scales": scales}
    if op == "linear":
        w = _mx4_values(t["codes"], t["scales"], case["K"])
        x = t["x"]
        if case["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * t["g"]
        return x @ w.t()
    if op == "write":
        _write_plain(t["kn"], t["kc"], t["ks"], t["pos"], t["n"])
        _write_plain(t["vn"], t["vc"], t["vs"], t["pos"], t["n"])
        return {"k": t["kc"], "v": t["vc"], "k_scale": t["ks"], "v_scale": t["vs"]}
    k = _cache_values(t["kc"], t["ks"], F32)
    v = _cache_values(t["vc"], t["vs"], F32)
    return _attend(t["q"].to(F32), k, v, t["lens"]).to(F16)


def _cache_values(codes, scales, dtype):
    B, G, L, D = codes.shape
    return (codes.to(dtype).view(B, G, L // KVB, KVB, D) * scales.to(dtype)[..., None, None]).view(B, G, L, D)


def _attend(q, k, v, lens):
    """softmax(q . k / sqrt(D)) . v over the first lens[b] tokens; zeros where there are none."""
    B, G, L, D = k.shape
    H = q.shape[1]
    s = torch.matmul(q.view(B, G, H // G, D), k.transpose(2, 3)) / math.sqrt(D)
    live = torch.arange(L, device=k.device) < lens.view(B, 1, 1, 1)
    s = torch.where(live, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(p, v).reshape(B, H, D)


def _write_plain(new, cache, scales, pos, n):
    """new [B, S, G, D] at tokens pos[b] .. pos[b] + n[b] - 1 of cache [B, G, room, D], in place."""
    B, S, G, D = new.shape
    nb = (S + KVB - 2) // KVB + 1  # blocks that S tokens can reach
    dev = new.device
    pos, n = pos.to(I64), n.to(I64)
    last = torch.div(pos + n - 1, KVB, rounding_mode="floor")
    blk = torch.div(pos, KVB, rounding_mode="floor")[:, None] + torch.arange(nb, device=dev)
    used = (blk <= last[:, None]) & (n > 0)[:, None]
    at = torch.where(used, blk, last[:, None]).clamp(0, scales.shape[2] - 1)
    bi = torch.arange(B, device=dev)[:, None].expand(B, nb)
    tok = at[:, :, None] * KVB + torch.arange(KVB, device=dev)
    fresh = (tok >= pos[:, None, None]) & (tok < (pos + n)[:, None, None])
    src = (tok - pos[:, None, None]).clamp(0, S - 1)
    x = new[bi[:, :, None].expand(src.shape), src].permute(0, 1, 3, 2, 4).to(F32)  # [B, nb, G, KVB, D]
    old = cache.view(U8).view(B, G, -1, KVB, D)[bi, :, at].view(F8).to(F32)
    s_old = scales[bi, :, at]
    fr = fresh[:, :, None, :, None]
    top = torch.where(fr & torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((-1, -2))
    kept = (at * KVB < pos[:, None])[:, :, None]
    s = _kv_scale(top)
    s = torch.where(kept, torch.maximum(s, s_old), s)
    r = (s_old / s)[..., None, None]
    before = (tok < pos[:, None, None])[:, :, None, :, None]
    val = torch.where(fr, x / s[..., None, None], torch.where(before, old * r, old)).to(F8)
    # a block named twice (the filling of `at`) gets the same bytes twice
    cache.view(U8).view(B, G, -1, KVB, D)[bi, :, at] = val.view(U8)
    scales[bi, :, at] = s


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "pack":
        n, es = case["rows"] * case["cols"], 2 if case["src"] == "f16" else 4
        packed = case["rows"] * -(-case["cols"] // MXB) * 17
        return {"bytes": 2 * n * es + 2 * packed, "flops": 2 * n}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * -(-K // MXB) * 17 + 4 * (M * K + M * N + (K if case["norm"] else 0)),
                "flops": 2 * M * N * K}
    B, G, D = case["batch"], case["kv_heads"], case["dim"]
    if op == "write":
        n = B * case["tokens"] * (0.75 if case["ragged"] and case["tokens"] > 1 else 1)
        return {"bytes": int(2 * n * G * D * 3), "flops": int(4 * n * G * D)}
    H, L = case["heads"], case["L"]
    tokens = B * L * (0.5 if case["ragged"] else 1)
    return {"bytes": int(2 * G * tokens * (D + 4 / KVB) + 4 * B * H * D), "flops": int(4 * H * tokens * D)}


# --------------------------------------------------------------------------
# results in 64 bits, from the definitions
# --------------------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx4_nearest64(x):
    """[rows, cols] -> (values, scale exponents): the nearest E2M1 value times the block's scale."""
    rows, cols = x.shape
    nb = -(-cols // MXB)
    p = torch.zeros((rows, nb * MXB), device=x.device, dtype=F64)
    p[:, :cols] = x.to(F64)
    p = p.view(rows, nb, MXB)
    top = p.abs().amax(-1)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.full_like(top, 2.0 ** -125)))) - 2
    scale = torch.pow(torch.full_like(e, 2.0), e.clamp(-127, 127)).unsqueeze(-1)
    m = p.abs() / scale
    best = torch.zeros_like(m)
    near = m.clone()
    for i, g in enumerate(_E2M1[1:], 1):
        dist = (m - g).abs()
        take = (dist < near) | ((dist == near) & (i % 2 == 0))
        best = torch.where(take, torch.full_like(best, g), best)
        near = torch.where(take, dist, near)
    return (torch.sign(p) * best * scale).view(rows, -1)[:, :cols], e.clamp(-127, 127)


def _mx4_value64(codes, scales, K):
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device, dtype=F64)
    rows = codes.shape[0]
    v = torch.empty((rows, codes.shape[1], 2), device=codes.device, dtype=F64)
    v[..., 0] = lut[(codes % 16).to(I64)]
    v[..., 1] = lut[(codes // 16).to(I64)]
    two = torch.full(scales.shape, 2.0, device=codes.device, dtype=F64)
    return (v.view(rows, -1, MXB) * torch.pow(two, scales.to(F64) - 127).unsqueeze(-1)).view(rows, -1)[:, :K]


def _append64(new, codes, scales, pos, n):
    """The cache after the write, sequence by sequence and block by block."""
    vals = codes.to(F64)
    sc = scales.to(F64)
    for b, (p, c) in enumerate(zip(pos.tolist(), n.tolist())):
        for blk in range(p // KVB, (p + c - 1) // KVB + 1 if c else 0):
            lo, hi = max(p, blk * KVB), min(p + c, (blk + 1) * KVB)
            x = new[b, lo - p:hi - p].to(F64).permute(1, 0, 2)  # [G, tokens, D]
            top = x.abs().amax((1, 2))
            e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 1e-9)) / 448))
            s = torch.pow(torch.full_like(e, 2.0), e.clamp(-15, 8))
            if lo > blk * KVB:
                s = torch.maximum(s, sc[b, :, blk])
                was = vals[b, :, blk * KVB:lo] * (sc[b, :, blk] / s)[:, None, None]
                vals[b, :, blk * KVB:lo] = was.to(F32).to(F8).to(F64)
            vals[b, :, lo:hi] = (x / s[:, None, None]).to(F32).to(F8).to(F64)
            sc[b, :, blk] = s
    return vals, sc


def exact(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    if op == "pack":
        v, e = _mx4_nearest64(t["W"])
        return {"values": v, "scales": (e + 127).to(U8)}
    if op == "linear":
        x = t["x"].to(F64)
        if case["norm"]:
            x = x * t["g"].to(F64) / torch.sqrt((x * x).sum(-1, keepdim=True) / case["K"] + EPS)
        return x @ _mx4_value64(t["codes"], t["scales"], case["K"]).t()
    if op == "write":
        k, ks = _append64(t["kn"], t["kc"], t["ks"], t["pos"], t["n"])
        v, vs = _append64(t["vn"], t["vc"], t["vs"], t["pos"], t["n"])
        return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}
    B, H, D = t["q"].shape
    G = case["kv_heads"]
    out = torch.zeros((B, H, D), device="cuda", dtype=F64)
    for b, n in enumerate(t["lens"].tolist()):
        if n:
            s = t["ks"][b].to(F64).repeat_interleave(KVB, 1)[:, :n, None]
            k = t["kc"][b, :, :n].to(F64) * s
            v = t["vc"][b, :, :n].to(F64) * t["vs"][b].to(F64).repeat_interleave(KVB, 1)[:, :n, None]
            q = t["q"][b].to(F64).view(G, H // G, D)
            w = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D), -1)
            out[b] = torch.matmul(w, v).view(H, D)
    return out
