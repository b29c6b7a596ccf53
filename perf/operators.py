"""The KV cache's operators, as cases to time and compare.

  store   kv_store then kv_load of the rows written: new k and v rows into a
          cache, and what the cache then holds for them
  load    kv_load: a range of cache rows read back as F32, per sequence
  attn    attn_kv: causal attention of the newest positions over a cache
  window  attn_kv with a sliding window and first rows that stay visible

A cache is F32, F16, BF16, or blocks of 32 values: Q8_0 {f16 d; i8 q[32]},
value q*d, and Q4_0 {f16 d; u8 q[16]}, the low nibbles values 0..15, the high
nibbles 16..31, value (nibble - 8)*d. `run` computes the plain form with
elementary torch operations in 32 bits, or, where `own` is true, calls the
framework.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "synthesize.cpp_amd")
_S = None

BLOCK = 32
BYTES = {"q8_0": 34, "q4_0": 18}
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _lib():
    global _S
    if _S is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import synth_hip
        _S = synth_hip
    return _S


def listed():
    return [
        # one token of one voice stream written at position 37: latency
        dict(name="store_token", kind="store", type="q4_0", n=1, t=1, cap=8192, kv=8, hd=128, ragged=False),
        # a batch of prompt chunks of unequal lengths, 16-bit cache
        dict(name="store_chunks_bf16", kind="store", type="bf16", n=5, t=509, cap=2048, kv=8, hd=128, ragged=True),
        # the longest prompt of the talker, one layer's rows
        dict(name="store_prompt_8192", kind="store", type="q4_0", n=1, t=8192, cap=8192, kv=8, hd=128, ragged=False),
        # a few prefixes of odd length read back (a cache taken up in another precision)
        dict(name="load_prefixes_q8", kind="load", type="q8_0", n=3, t=1021, cap=2048, kv=8, hd=128, ragged=True),
        # the whole caches of sixteen long sequences
        dict(name="load_16x8192", kind="load", type="q4_0", n=16, t=8192, cap=8192, kv=8, hd=128, ragged=False),
        # a voice stream's first frames: one query, 38 rows, latency
        dict(name="decode_38", kind="attn", type="q4_0", n=1, t=1, cap=38, heads=16, kv=8, hd=128, ragged=False),
        # the end of the longest single stream
        dict(name="decode_8191", kind="attn", type="q4_0", n=1, t=1, cap=8191, heads=16, kv=8, hd=128, ragged=False),
        # 64 concurrent streams of different lengths
        dict(name="decode_64_streams", kind="attn", type="q4_0", n=64, t=1, cap=8192, heads=16, kv=8, hd=128,
             ragged=True),
        # an ordinary prompt of odd length over an 8-bit cache
        dict(name="prefill_1021_q8", kind="attn", type="q8_0", n=1, t=1021, cap=1021, heads=16, kv=8, hd=128,
             ragged=False),
        # the longest prompt
        dict(name="prefill_8192", kind="attn", type="q4_0", n=1, t=8192, cap=8192, heads=16, kv=8, hd=128,
             ragged=False),
        # long-running streams kept to a window of 1000 rows and 4 first ones
        dict(name="window_decode_32", kind="window", type="q4_0", n=32, t=1, cap=8192, heads=16, kv=8, hd=128,
             window=1000, sinks=4, ragged=True),
        # a long prompt under the same kind of mask
        dict(name="window_prefill_8192", kind="window", type="q4_0", n=1, t=8192, cap=8192, heads=16, kv=8, hd=128,
             window=1024, sinks=4, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "load", "attn", "attn", "window", "window"])
    kind_type = rng.choice(["q4_0", "q4_0", "q8_0", "f16", "bf16", "f32"])
    hd = rng.choice([64, 96, 128, 128]) if kind_type in BYTES else rng.choice([40, 64, 80, 96, 128])
    kv, group = rng.choice([(8, 2), (8, 1), (4, 4), (2, 7), (1, 8), (12, 1), (2, 16)])
    n = _log(rng, 1, 64)
    c = dict(kind=kind, type=kind_type, n=n, kv=kv, hd=hd, ragged=rng.choice([False, True]))
    if kind in ("store", "load"):
        c["t"] = _log(rng, 1, max(1, min(8192, 65536 // n)))
        c["cap"] = c["t"] + rng.randrange(0, 600)
        return c
    c["heads"] = kv * group
    if rng.random() < 0.5:  # decoding: one position, or a few checked at once
        c["t"] = rng.choice([1, 1, 1, 2, 5])
        c["cap"] = c["t"] + _log(rng, 1, max(2, min(16000, 200000 // n)))
    else:  # a prompt, or a chunk of one behind earlier rows
        c["n"] = n = min(n, 8)
        c["t"] = _log(rng, 16, max(17, 4096 // n))
        c["cap"] = c["t"] + rng.choice([0, rng.randrange(1, 2000)])
    if kind == "window":
        c["window"] = _log(rng, 2, 3000)
        c["sinks"] = rng.choice([0, 1, 4, 4, 67])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _pack(x, kind):
    """A cache tensor (..., hd) F32 in its storage type (blocks as uint8)."""
    if kind in FLOAT:
        return x.to(FLOAT[kind])
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    mag = b.abs()
    top = mag.amax(-1, keepdim=True)
    if kind == "q8_0":
        d = (top.double() / 127.0).float()
    else:  # the first value of the largest magnitude, with its sign, becomes -8
        lane = torch.arange(BLOCK, device=x.device)
        first = torch.where(mag == top, lane, BLOCK).amin(-1, keepdim=True)
        d = b.gather(-1, first) / -8.0
    inv = torch.where(d.abs() >= 2.0 ** -126, 1.0 / d.double(), 0.0).float()
    v = b * inv
    if kind == "q8_0":
        whole = v.trunc()
        q = whole + torch.where((v - whole).abs() >= 0.5, v.sign(), 0.0)
        q = q.to(torch.int8).view(torch.uint8)
    else:
        q = (v + 8.5).trunc().clamp(max=15.0).to(torch.uint8)
        q = q[..., :16] | (q[..., 16:] << 4)
    return torch.cat([d.to(torch.float16).view(torch.uint8), q], -1).flatten(-2)


def _unpack(c, kind):
    """The F32 values (..., hd) that a cache tensor stands for."""
    if kind in FLOAT:
        return c.float()
    b = c.unflatten(-1, (-1, BYTES[kind]))
    d = b[..., :2].contiguous().view(torch.float16).float()
    q = b[..., 2:]
    if kind == "q8_0":
        q = q.contiguous().view(torch.int8).float()
    else:
        q = torch.cat([q & 15, q >> 4], -1).float() - 8.0
    return (q * d).flatten(-2)


def _row(case):
    """The last extent of a cache tensor as torch holds it."""
    return case["hd"] // BLOCK * BYTES[case["type"]] if case["type"] in BYTES else case["hd"]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def some(low, high):  # one whole number of [low, high] for each sequence
        return torch.randint(low, high + 1, (n,), generator=g, device="cuda", dtype=torch.int32)

    n, t, cap, kv, hd, ragged = (case[k] for k in ("n", "t", "cap", "kv", "hd", "ragged"))
    s = dict(case)
    s["count"] = some(max(0, t // 3), t) if ragged and (t > 1 or case["kind"] in ("store", "load")) else None
    # normalised keys have a few strong channels; values are smaller
    gain = 1.0 + 2.0 * (torch.rand(hd, generator=g, device="cuda") < 0.05)
    if case["kind"] == "store":
        s["x"] = [randn(n, t, kv, hd) * gain, 0.5 * randn(n, t, kv, hd)]
        s["slot"] = some(0, cap - t)
        kind = FLOAT.get(case["type"], torch.uint8)
        s["cache"] = [torch.zeros(n, cap, kv, _row(case), dtype=kind, device="cuda") for _ in range(2)]
        s["out"] = [torch.zeros(n, t, kv, hd, device="cuda") for _ in range(2)]
        return s
    s["cache"] = [_pack(randn(n, cap, kv, hd) * gain, case["type"]), _pack(0.5 * randn(n, cap, kv, hd), case["type"])]
    if case["kind"] == "load":
        s["slot"] = some(0, cap - t)
        s["out"] = [torch.zeros(n, t, kv, hd, device="cuda") for _ in range(2)]
        return s
    s["q"] = 1.5 * randn(n, t, case["heads"], hd)
    s["length"] = some(max(t, cap // 16), cap) if ragged else some(cap, cap)
    s["scale"] = 1.0 / math.sqrt(hd)
    s["window"], s["sinks"] = case.get("window", 0), case.get("sinks", 0)
    s["y"] = torch.zeros(n, t, case["heads"], hd, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"store": _store, "load": _load}.get(state["kind"], _attend)(state)


def _run_own(s):
    S = _lib()
    caches = s["cache"]
    if s["type"] in BYTES:
        cls = S.Q8Tensor if s["type"] == "q8_0" else S.Q4Tensor
        caches = [cls(c, s["hd"]) for c in caches]
    if s["kind"] == "store":
        S.kv_store(s["x"][0], s["x"][1], caches[0], caches[1], s["slot"], s["count"])
    if s["kind"] in ("store", "load"):
        return S.kv_load(caches[0], caches[1], s["slot"], s["t"], s["count"], k_out=s["out"][0], v_out=s["out"][1])
    return S.attn_kv(s["q"], caches[0], caches[1], s["length"], s["count"], scale=s["scale"], window=s["window"],
                     sinks=s["sinks"], out=s["y"])


def _live(s, rows):
    """(n, t, 1, 1): whether query or row t of sequence n is one, or padding."""
    return None if s["count"] is None else (rows[None, :] < s["count"][:, None])[..., None, None]


def _store(s):
    rows = torch.arange(s["t"], device="cuda")
    seq = torch.arange(s["n"], device="cuda")[:, None]
    at = s["slot"][:, None] + rows
    live = _live(s, rows)
    for x, cache in zip(s["x"], s["cache"]):
        new = _pack(x, s["type"])
        cache[seq, at] = new if live is None else torch.where(live, new, cache[seq, at])
    return _load(s)


def _load(s):
    rows = torch.arange(s["t"], device="cuda")
    seq = torch.arange(s["n"], device="cuda")[:, None]
    at = s["slot"][:, None] + rows
    live = _live(s, rows)
    got = [_unpack(cache[seq, at], s["type"]) for cache in s["cache"]]
    return got if live is None else [torch.where(live, x, o) for x, o in zip(got, s["out"])]


def _attend(s):
    n, t, heads, hd = s["q"].shape
    kv = s["kv"]
    k, v = (_unpack(c, s["type"]).transpose(1, 2).contiguous() for c in s["cache"])  # (n, kv, cap, hd)
    q = s["q"].reshape(n, t, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"]).view(n, kv, heads // kv, t, -1)
    rows = torch.arange(t, device="cuda")
    keys = torch.arange(k.shape[2], device="cuda")
    count = s["count"] if s["count"] is not None else torch.full_like(s["length"], t)
    at = ((s["length"] - count)[:, None] + rows)[:, :, None]  # (n, t, 1)
    seen = keys <= at
    if s["window"]:
        seen &= (keys > at - s["window"]) | (keys < s["sinks"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(n, kv, -1, p.shape[-1]), v).view(n, kv, heads // kv, t, hd)
    y = y / torch.where(total == 0.0, 1.0, total)
    y = y.permute(0, 3, 1, 2, 4).reshape(n, t, heads, hd)
    live = _live(s, rows)
    return y if live is None else torch.where(live, y, s["y"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def _mean_count(case):
    """The expected number of real rows of a sequence."""
    t = case["t"]
    if not case["ragged"] or (t == 1 and case["kind"] in ("attn", "window")):
        return float(t)
    return (max(0, t // 3) + t) / 2.0


def work(case):
    n, t, cap, kv, hd = (case[k] for k in ("n", "t", "cap", "kv", "hd"))
    value = BYTES[case["type"]] / BLOCK if case["type"] in BYTES else FLOAT[case["type"]].itemsize
    rows = n * _mean_count(case)
    row = kv * hd
    if case["kind"] == "store":  # F32 in, the cache written and read, F32 out; about ten operations a value
        return {"bytes": 2 * rows * row * (4 + 2 * value + 4), "flops": 2 * rows * row * 10}
    if case["kind"] == "load":
        return {"bytes": 2 * rows * row * (value + 4), "flops": 2 * rows * row * 2}
    length = (max(t, cap // 16) + cap) / 2.0 if case["ragged"] else float(cap)
    c = _mean_count(case)
    window, sinks = case.get("window", 0), case.get("sinks", 0)

    def mean_seen(p):  # rows seen from position p
        if not window or p + 1 <= window:
            return p + 1
        return window + min(sinks, p + 1 - window)

    steps = 64
    seen = sum(mean_seen(length - c + c * (i + 0.5) / steps) for i in range(steps)) / steps if c > 1 else \
        mean_seen(length - 1)
    first = length - c
    touched = length if not window else min(length, c - 1 + window + min(sinks, max(0.0, first + 1 - window)))
    return {"bytes": n * (2 * touched * row * value + 2 * c * case["heads"] * hd * 4),
            "flops": 4.0 * n * c * case["heads"] * hd * seen}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _values64(c, case):
    """What a cache tensor's rows stand for, in 64 bits: block by block."""
    if case["type"] in FLOAT:
        return c.double()
    size = BYTES[case["type"]]
    blocks = c.reshape(-1, size)
    d = blocks[:, 0:2].contiguous().view(torch.float16).double()
    out = torch.empty(blocks.shape[0], BLOCK, dtype=torch.float64, device=c.device)
    if case["type"] == "q8_0":
        code = blocks[:, 2:].to(torch.float64)
        out[:] = torch.where(code > 127, code - 256, code) * d
    else:
        code = blocks[:, 2:].to(torch.float64)
        high = torch.floor(code / 16)
        out[:, :16] = (code - 16 * high - 8) * d
        out[:, 16:] = (high - 8) * d
    return out.reshape(*c.shape[:-1], case["hd"])


def _rounded64(x, case):
    """The values that the cache holds for x: F16 and BF16 by rounding, blocks by
    the codes' formula, whose products, sums and quotients are rounded to 32 bits."""
    if case["type"] in FLOAT:
        return x.to(FLOAT[case["type"]]).double()
    b = x.reshape(-1, BLOCK)
    hi, lo = b.max(1, keepdim=True).values, b.min(1, keepdim=True).values
    if case["type"] == "q8_0":
        d = (torch.maximum(hi, -lo).double() / 127).float()
    else:
        place = torch.arange(BLOCK, device=b.device).expand_as(b)
        at_hi = place.masked_fill(b != hi, BLOCK).min(1, keepdim=True).values
        at_lo = place.masked_fill(b != lo, BLOCK).min(1, keepdim=True).values
        positive = (hi > -lo) | ((hi == -lo) & (at_hi < at_lo))
        d = torch.where(positive, hi, lo) * -0.125
    inv = torch.where(d.double().abs() < 2.0 ** -126, 0.0, 1 / d.double()).float()
    v = (b.double() * inv.double()).float()
    if case["type"] == "q8_0":
        code = torch.floor(v.double().abs() + 0.5) * torch.sign(v.double())
    else:
        code = torch.floor((v.double() + 8.5).float().double()).clamp(0, 15) - 8
    return (code * d.half().double()).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    n, t = case["n"], case["t"]
    if case["kind"] in ("store", "load"):
        out = []
        for i in range(2):
            y = s["out"][i].double()
            for b in range(n):
                c = t if s["count"] is None else int(s["count"][b])
                at = int(s["slot"][b])
                y[b, :c] = _rounded64(s["x"][i][b, :c], case) if case["kind"] == "store" else \
                    _values64(s["cache"][i][b, at:at + c], case)
            out.append(y)
        return out
    y = s["y"].double()
    group = case["heads"] // case["kv"]
    for b in range(n):
        length = int(s["length"][b])
        c = t if s["count"] is None else int(s["count"][b])
        k, v = (_values64(x[b, :length], case) for x in s["cache"])
        p = (length - c + torch.arange(c, device="cuda"))[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = j > p
        if s["window"]:
            hidden |= (p - j >= s["window"]) & (j >= s["sinks"])
        for h in range(case["heads"]):
            w = s["scale"] * (s["q"][b, :c, h].double() @ k[:, h // group].T)
            w = torch.softmax(w.masked_fill(hidden, -math.inf), 1)
            y[b, :c, h] = w @ v[:, h // group]
    return y
