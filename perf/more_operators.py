"""The paged KV cache's operators and the attention to an encoder, as cases to
time and compare.

  pages   kv_pages and kv_slots: the pages of sequences that arrive, grow and end,
          the slots of their new rows, and the step that takes all of it back
  store   kv_store_pages then kv_load_pages of every row of the pages written
  attn    attn_pages: causal attention of the newest positions over a paged cache,
          whole or through a window with first rows that stay visible
  cross   attn_cross: attention of all queries to all of an encoder's states

A paged cache has blocks of `page` positions of one head, int8 codes under one F32
scale: a value is code * scale. K's blocks are [page][hd], V's [hd][page]; row r
of a sequence is row r % page of the page that its table names at r / page. `run`
computes the plain form with elementary torch operations in 32 bits, or, where
`own` is true, calls the framework.
"""
import math
import os
import sys

import numpy
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "synthesize.cpp_amd")
_S = None

FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
I32 = torch.int32


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
        # one decoding step of 64 voice streams, some of which begin a page: latency
        dict(name="pages_step_64", kind="pages", n=64, page=16, cap=8192, t=1),
        # a busy server's step: 2048 requests, of which some arrive with a prompt and some end
        dict(name="pages_admit_2048", kind="pages", n=2048, page=16, cap=4096, t=509),
        # one token of one stream, inside a page that has earlier rows
        dict(name="store_token", kind="store", n=1, t=1, cap=8192, page=64, kv=8, hd=128, ragged=False),
        # chunks of prompts of unequal lengths that begin and end inside pages
        dict(name="store_chunks", kind="store", n=5, t=509, cap=2048, page=32, kv=8, hd=128, ragged=True),
        # the longest prompt of the talker, one layer's rows
        dict(name="store_prompt_8192", kind="store", n=1, t=8192, cap=8192, page=64, kv=8, hd=128, ragged=False),
        # a voice stream's first frames: one query, 38 rows, latency
        dict(name="decode_38", kind="attn", n=1, t=1, cap=38, page=16, heads=16, kv=8, hd=128, ragged=False),
        # 64 concurrent streams of different lengths
        dict(name="decode_64_streams", kind="attn", n=64, t=1, cap=8192, page=64, heads=16, kv=8, hd=128, ragged=True),
        # an ordinary prompt of odd length
        dict(name="prefill_1021", kind="attn", n=1, t=1021, cap=1021, page=64, heads=16, kv=8, hd=128, ragged=False),
        # the longest prompt
        dict(name="prefill_8192", kind="attn", n=1, t=8192, cap=8192, page=64, heads=16, kv=8, hd=128, ragged=False),
        # a decoder's token of sixteen streams against encoded texts or voices of different lengths
        dict(name="cross_token_f16", kind="cross", type="f16", n=16, t=1, rows=1500, heads=16, kv=16, hd=64, ragged=True),
        # a text encoder's layer: every phoneme sees every other
        dict(name="cross_text_510", kind="cross", type="f32", n=4, t=510, rows=510, heads=12, kv=12, hd=64, ragged=False),
        # a long target against a long source
        dict(name="cross_4096_bf16", kind="cross", type="bf16", n=2, t=4096, rows=1500, heads=16, kv=8, hd=128,
             ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "store", "attn", "attn", "attn", "cross", "cross"])
    if kind == "pages":
        n, cap = _log(rng, 1, 2048), _log(rng, 64, 8192)
        return dict(kind=kind, n=n, page=rng.choice([16, 32, 64, 128]), cap=cap,
                    t=rng.choice([1, _log(rng, 2, max(3, min(cap, 600000 // n)))]))
    c = dict(kind=kind, n=_log(rng, 1, 64), ragged=rng.choice([False, True]))
    if kind == "cross":
        c["type"] = rng.choice(["f32", "f16", "bf16"])
        c["kv"], group = rng.choice([(16, 1), (12, 1), (8, 2), (4, 4), (2, 7)])
        c["hd"] = rng.choice([40, 64, 64, 80, 96, 128])
        c["heads"] = c["kv"] * group
        c["rows"] = _log(rng, 1, 3000)
        if rng.random() < 0.5:
            c["t"] = rng.choice([1, 1, 2, 5])
        else:
            c["n"] = min(c["n"], 8)
            c["t"] = _log(rng, 8, max(9, 8192 // c["n"]))
        return c
    c["page"] = rng.choice([16, 32, 64, 64, 128])
    c["hd"] = rng.choice([64, 80, 96, 128, 128])
    c["kv"], group = rng.choice([(8, 2), (8, 1), (4, 4), (2, 7), (1, 8), (12, 1), (2, 16)])
    n = c["n"]
    if kind == "store":
        c["t"] = _log(rng, 1, max(1, min(8192, 65536 // n)))
        c["cap"] = c["t"] + rng.randrange(0, 600)
        return c
    c["heads"] = c["kv"] * group
    if rng.random() < 0.5:  # decoding: one position, or a few checked at once
        c["t"] = rng.choice([1, 1, 1, 2, 5])
        c["cap"] = c["t"] + _log(rng, 1, max(2, min(16000, 200000 // n)))
    else:  # a prompt, or a chunk of one behind earlier rows
        c["n"] = n = min(n, 8)
        c["t"] = _log(rng, 16, max(17, 4096 // n))
        c["cap"] = c["t"] + rng.choice([0, rng.randrange(1, 2000)])
    if rng.random() < 0.4:
        c["window"] = _log(rng, 2, 3000)
        c["sinks"] = rng.choice([0, 1, 4, 4, 67])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, t = case["n"], case["t"]
    s = dict(case)

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def some(low, high):  # one whole number of [low, high] for each sequence
        return torch.randint(low, high + 1, (n,), generator=g, device="cuda", dtype=I32)

    if case["kind"] == "cross":
        kv, hd, rows = case["kv"], case["hd"], case["rows"]
        gain = 1.0 + 2.0 * (rand(hd) < 0.05)
        s["q"] = 1.5 * randn(n, t, case["heads"], hd)
        s["k"] = (randn(n, rows, kv, hd) * gain).to(FLOAT[case["type"]])
        s["v"] = (0.5 * randn(n, rows, kv, hd)).to(FLOAT[case["type"]])
        s["length"] = some(max(1, rows // 5), rows) if case["ragged"] else None
        s["count"] = some(max(1, t // 3), t) if case["ragged"] and t > 1 else None
        s["scale"] = 1.0 / math.sqrt(hd)
        s["y"] = torch.zeros(n, t, case["heads"], hd, device="cuda")
        return s

    page, cap = case["page"], case["cap"]
    most = (cap + page - 1) // page  # pages of the longest sequence
    if case["kind"] == "pages":
        # before: most requests run, some places are empty. After: running ones have
        # one row more or (a few) have ended, and empty places are taken by prompts
        before = torch.where(rand(n) < 0.15, 0, some(1, max(1, cap - t)))
        prompt = torch.where(rand(n) < 0.5, some(max(1, t // 3), t), 0)
        after = torch.where(before == 0, prompt, torch.where(rand(n) < 0.1, 0, (before + 1).clamp(max=cap)))
        s["before"], s["after"] = before.to(I32), after.to(I32)
        s["count"] = (s["after"] - s["before"]).clamp(min=0).to(I32)
        held = (s["before"] + page - 1) // page
        order = torch.randperm(n * most, generator=g, device="cuda").to(I32)
        used = torch.arange(most, device="cuda") < held[:, None]
        s["table"] = torch.where(used, order.view(n, most), -1)
        spare = order[~used.flatten()]
        s["free"] = torch.full((n * most,), -1, dtype=I32, device="cuda")
        s["free"][:spare.numel()] = spare
        s["left"] = torch.tensor([spare.numel()], dtype=I32, device="cuda")
        s["held"] = held.to(I32)
        s["slots"] = torch.zeros(n, t, dtype=I32, device="cuda")
        return s

    kv, hd, ragged = case["kv"], case["hd"], case["ragged"]
    pages = n * most + 1  # the last is in no table
    gain = 1.0 + 2.0 * (rand(hd) < 0.05)  # normalised keys have a few strong channels; values are smaller

    def codes(row, spread):  # of blocks whose largest magnitude is about 3.5 of the strongest channel's deviations
        x = torch.randn((pages, kv, page, hd), generator=g, device="cuda", dtype=torch.float16)
        x = x.mul_((row * (127.0 / 3.5 / spread)).half()).round_().clamp_(-127, 127).to(torch.int8)
        return x, (3.5 * spread / 127.0) * (0.5 + rand(pages, kv))

    s["k"], s["k_scale"] = codes(gain, 3.0)
    v, s["v_scale"] = codes(torch.ones(hd, device="cuda"), 1.0)
    s["v"] = v.transpose(2, 3).contiguous()
    s["v_scale"] *= 0.5
    s["table"] = torch.randperm(pages - 1, generator=g, device="cuda").to(I32).view(n, most)
    if case["kind"] == "store":
        s["count"] = some(max(0, t // 3), t) if ragged else None
        start = some(0, cap - t)
        count = s["count"] if s["count"] is not None else torch.full_like(start, t)
        s["length"] = start + count
        s["x"] = [randn(n, t, kv, hd) * gain, 0.5 * randn(n, t, kv, hd)]
        # every row of the first page written, and on to the last new one
        first = start - start % page
        at = first[:, None] + torch.arange(t + page - 1, device="cuda", dtype=I32)
        slot = s["table"].gather(1, (at // page).clamp(max=most - 1).long()) * page + at % page
        s["slots"] = torch.where(at < s["length"][:, None], slot, -1).to(I32)
        s["out"] = [torch.zeros(n, t + page - 1, kv, hd, device="cuda") for _ in range(2)]
        return s
    s["count"] = some(max(0, t // 3), t) if ragged and t > 1 else None
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
    return {"pages": _pages, "store": _store, "attn": _attend, "cross": _cross}[state["kind"]](state)


def _run_own(s):
    S = _lib()
    if s["kind"] == "cross":
        return S.attn_cross(s["q"], s["k"], s["v"], s["length"], s["count"], scale=s["scale"], out=s["y"])
    if s["kind"] == "pages":
        S.kv_pages(s["after"], s["page"], s["held"], s["free"], s["left"], s["table"])
        S.kv_slots(s["table"], s["after"], s["page"], s["t"], s["count"], out=s["slots"])
        S.kv_pages(s["before"], s["page"], s["held"], s["free"], s["left"], s["table"])
        return [s["slots"], s["table"], s["held"], s["left"]]
    cache = S.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["kind"] == "store":
        S.kv_store_pages(s["x"][0], s["x"][1], cache, s["table"], s["length"], s["count"])
        out = S.kv_load_pages(cache, s["slots"], k_out=s["out"][0], v_out=s["out"][1])
        return [*out, s["k_scale"], s["v_scale"]]
    return S.attn_pages(s["q"], cache, s["table"], s["length"], s["count"], scale=s["scale"], window=s["window"],
                        sinks=s["sinks"], out=s["y"])


def _fit(s, length):
    """Tables for new lengths: pages past a sequence's need go back on the stack
    of free ones, the last of the last sequence first; then missing ones are taken
    from its top, the first of the first sequence first."""
    need = (length + s["page"] - 1) // s["page"]
    held, table, left = s["held"][:, None], s["table"], s["left"]
    col = torch.arange(table.shape[1], device="cuda")
    back = (col >= need[:, None]) & (col < held)
    take = (col < need[:, None]) & (col >= held)
    number = back.flatten().cumsum(0).view_as(back)
    total = left + number[-1, -1]
    spare = torch.cat([s["free"], s["free"][:1]])  # (a place for what is not given back)
    spare[torch.where(back, total - number, spare.numel() - 1)] = table
    s["free"].copy_(spare[:-1])
    number = take.flatten().cumsum(0).view_as(take)
    table.copy_(torch.where(take, s["free"][(total - number).clamp(0, s["free"].numel() - 1)], torch.where(back, -1, table)))
    s["left"].copy_(total - number[-1, -1])
    s["held"].copy_(need)


def _pages(s):
    _fit(s, s["after"])
    t = torch.arange(s["t"], device="cuda", dtype=I32)
    at = (s["after"] - s["count"])[:, None] + t
    page = s["table"].gather(1, (at // s["page"]).clamp(0, s["table"].shape[1] - 1).long())
    s["slots"].copy_(torch.where(t < s["count"][:, None], page * s["page"] + at % s["page"], -1))
    _fit(s, s["before"])
    return [s["slots"], s["table"], s["held"], s["left"]]


def _live(s, rows):
    """(n, t, 1, 1): whether query or row t of sequence n is one, or padding."""
    return None if s["count"] is None else (rows[None, :] < s["count"][:, None])[..., None, None]


def _store(s):
    n, t, kv, hd = s["x"][0].shape
    page, table = s["page"], s["table"]
    count = s["count"] if s["count"] is not None else torch.full_like(s["length"], t)
    start = (s["length"] - count)[:, None]
    unit = start // page + torch.arange((t + page - 2) // page + 1, device="cuda")
    at = unit[..., None] * page + torch.arange(page, device="cuda")  # (n, units, page): the blocks' rows
    new = (at >= start[..., None]) & (at < s["length"][:, None, None])
    last = s["k"].shape[0] - 1
    where = torch.where(new.any(-1), table.gather(1, unit.clamp(max=table.shape[1] - 1)), last).long()
    row = (at - start[..., None]).clamp(0, t - 1).flatten(1)
    seq = torch.arange(n, device="cuda")[:, None]
    had = (unit * page < start)[..., None]
    for x, codes, scale in zip(s["x"], (s["k"], s["v"]), (s["k_scale"], s["v_scale"])):
        old = codes[where]
        old = (old if codes is s["k"] else old.transpose(3, 4)).float()  # (n, units, kv, page, hd)
        fresh = x[seq, row].view(n, -1, page, kv, hd).transpose(2, 3)
        is_new = new[:, :, None, :, None]
        d_old = scale[where]
        d = torch.where(is_new, fresh.abs(), 0.0).amax((3, 4)) / 127.0
        d = torch.where(had, torch.maximum(d, d_old), d)
        d = torch.where(new.any(-1)[..., None], d, d_old)
        by = torch.where(d > d_old, d_old / d, 1.0)[..., None, None]
        kept = (old * by).round()
        made = (fresh / d[..., None, None]).round().clamp(-127.0, 127.0)
        c = torch.where(is_new, torch.where(d[..., None, None] == 0.0, 0.0, made), torch.where(had[..., None, None], kept, old))
        c = c.to(torch.int8)
        codes[where] = c if codes is s["k"] else c.transpose(3, 4)
        scale[where] = d
    # the rows read back
    slot = s["slots"].clamp(min=0).long()
    live = (s["slots"] >= 0)[..., None, None]
    k = s["k"][slot // page, :, slot % page].float() * s["k_scale"][slot // page][..., None]
    v = s["v"][slot // page, :, :, slot % page].float() * s["v_scale"][slot // page][..., None]
    return [torch.where(live, k, s["out"][0]), torch.where(live, v, s["out"][1]), s["k_scale"], s["v_scale"]]


def _softmax_sum(q, k, v, seen, scale):
    """q (n, t, heads, hd), k and v (n, kv, rows, hd), seen (n or 1, t or 1, rows)."""
    n, t, heads, hd = q.shape
    kv = k.shape[1]
    q = q.reshape(n, t, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).view(n, kv, heads // kv, t, -1)
    if seen is not None:
        scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(n, kv, -1, p.shape[-1]), v).view(n, kv, heads // kv, t, hd)
    y = y / torch.where(total == 0.0, 1.0, total)
    return y.permute(0, 3, 1, 2, 4).reshape(n, t, heads, hd)


def _attend(s):
    n, t, heads, hd = s["q"].shape
    table = s["table"].long()
    k = s["k"][table].float() * s["k_scale"][table][..., None, None]  # (n, pages, kv, page, hd)
    k = k.transpose(1, 2).reshape(n, s["kv"], -1, hd)
    v = s["v"][table].float() * s["v_scale"][table][..., None, None]  # (n, pages, kv, hd, page)
    v = v.permute(0, 2, 1, 4, 3).reshape(n, s["kv"], -1, hd)
    rows = torch.arange(t, device="cuda")
    keys = torch.arange(k.shape[2], device="cuda")
    count = s["count"] if s["count"] is not None else torch.full_like(s["length"], t)
    at = ((s["length"] - count)[:, None] + rows)[:, :, None]  # (n, t, 1)
    seen = keys <= at
    if s["window"]:
        seen &= (keys > at - s["window"]) | (keys < s["sinks"])
    y = _softmax_sum(s["q"], k, v, seen, s["scale"])
    live = _live(s, rows)
    return y if live is None else torch.where(live, y, s["y"])


def _cross(s):
    k, v = (x.float().transpose(1, 2).contiguous() for x in (s["k"], s["v"]))
    keys = torch.arange(s["rows"], device="cuda")
    seen = None if s["length"] is None else (keys < s["length"][:, None])[:, None]
    y = _softmax_sum(s["q"], k, v, seen, s["scale"])
    live = _live(s, torch.arange(s["t"], device="cuda"))
    return y if live is None else torch.where(live, y, s["y"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def _mean_count(case):
    """The expected number of real rows of a sequence."""
    t = case["t"]
    if not case["ragged"] or (t == 1 and case["kind"] != "store"):
        return float(t)
    return (max(1 if case["kind"] == "cross" else 0, t // 3) + t) / 2.0


def work(case):
    n, t = case["n"], case["t"]
    if case["kind"] == "pages":
        # lengths and pages held, read and written; a table entry and a place of the
        # stack for every page that changes hands, both ways; the slots
        mean = (1 + max(1, case["cap"] - t)) / 2.0
        pages = n * (0.85 * (0.1 * mean + 0.9) + 0.15 * 0.5 * (t // 3 + t) / 2.0) / case["page"]
        return {"bytes": n * 4 * 8 + 2 * pages * 4 * 4 + n * t * 4, "flops": n * t * 4 + 2 * pages * 8}
    hd, kv = case["hd"], case["kv"]
    rows = n * _mean_count(case)
    if case["kind"] == "store":  # F32 in, a byte written and read, F32 out; about ten operations a value
        values = 2.0 * rows * kv * hd
        return {"bytes": values * (4 + 1 + 1 + 4), "flops": values * 10}
    c, heads = _mean_count(case), case["heads"]
    qy = 2 * n * c * heads * hd * 4
    if case["kind"] == "cross":
        length = (max(1, case["rows"] // 5) + case["rows"]) / 2.0 if case["ragged"] else float(case["rows"])
        return {"bytes": n * 2 * length * kv * hd * FLOAT[case["type"]].itemsize + qy,
                "flops": 4.0 * n * c * heads * hd * length}
    cap = case["cap"]
    length = (max(t, cap // 16) + cap) / 2.0 if case["ragged"] else float(cap)
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
    return {"bytes": n * 2 * touched * kv * (hd + 4.0 / case["page"]) + qy, "flops": 4.0 * n * c * heads * hd * seen}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "store": _exact_store, "attn": _exact_attend, "cross": _exact_cross}[case["kind"]](s)


def _exact_pages(s):
    """Request by request, with a list for the stack."""
    page = s["page"]
    stack = s["free"][:int(s["left"])].tolist()
    own_pages = [[p for p in row if p >= 0] for row in s["table"].tolist()]

    def fit(lengths):
        for pages, length in reversed(list(zip(own_pages, lengths))):
            while len(pages) > -(-length // page):
                stack.append(pages.pop())
        for pages, length in zip(own_pages, lengths):
            while len(pages) < -(-length // page):
                pages.append(stack.pop())

    after, count = s["after"].tolist(), s["count"].tolist()
    fit(after)
    slots = numpy.full((s["n"], s["t"]), -1, dtype=numpy.int32)
    for b, pages in enumerate(own_pages):
        if count[b]:
            r = numpy.arange(after[b] - count[b], after[b])
            slots[b, :count[b]] = numpy.asarray(pages)[r // page] * page + r % page
    fit(s["before"].tolist())
    table = [row + [-1] * (s["table"].shape[1] - len(row)) for row in own_pages]

    def out(x):
        return torch.tensor(x, dtype=I32, device="cuda")

    return [out(slots), out(table), out([len(row) for row in own_pages]), out([len(stack)])]


def _exact_store(s):
    """Page by page. The codes are defined by quotients and products that are
    rounded to 32 bits; those of two 32-bit numbers in 64 bits round as they do."""
    page, t = s["page"], s["t"]
    scales = [s["k_scale"].double(), s["v_scale"].double()]
    values = [x.double() for x in s["out"]]
    for b in range(s["n"]):
        length = int(s["length"][b])
        count = t if s["count"] is None else int(s["count"][b])
        start = length - count
        if count == 0:
            rows = range(start - start % page, length)
            pages = range(start // page, (length + page - 1) // page)
        else:
            rows = range(start - start % page, length)
            pages = range(start // page, (length - 1) // page + 1)
        for i in pages:
            where = int(s["table"][b, i])
            lo, hi = max(start, i * page), min(length, (i + 1) * page)
            for side, pool in enumerate((s["k"], s["v"].transpose(2, 3))):
                d_old = scales[side][where].clone()                   # (kv,)
                older = pool[where, :, :max(0, lo - i * page)].double()  # (kv, rows, hd)
                x = s["x"][side][b, lo - start:hi - start].double().transpose(0, 1)
                d = d_old
                if count:
                    d = (x.abs().flatten(1).max(1).values / 127).float().double()
                    if lo > i * page:
                        d = torch.maximum(d, d_old)
                    by = torch.where(d > d_old, (d_old / d).float().double(), 1.0)
                    older = torch.round((older * by[:, None, None]).float().double())
                scales[side][where] = d
                fresh = torch.round((x / d[:, None, None]).float().double()).clamp(-127, 127)
                fresh = torch.where(d[:, None, None] == 0, 0.0, fresh)
                first = i * page - rows[0] if len(rows) else 0
                got = torch.cat([older, fresh], 1) * d[:, None, None]
                values[side][b, first:first + got.shape[1]] = got.transpose(0, 1)
    return [*values, *scales]


def _weigh(s, y, b, c, k, v, hidden):
    group = s["heads"] // s["kv"]
    for h in range(s["heads"]):
        w = s["scale"] * (s["q"][b, :c, h].double() @ k[h // group].T)
        if hidden is not None:
            w = w.masked_fill(hidden, -math.inf)
        y[b, :c, h] = torch.softmax(w, 1) @ v[h // group]


def _exact_attend(s):
    y = s["y"].double()
    for b in range(s["n"]):
        length = int(s["length"][b])
        c = s["t"] if s["count"] is None else int(s["count"][b])
        of = s["table"][b, :(length + s["page"] - 1) // s["page"]].long()
        k = s["k"][of].double() * s["k_scale"][of].double()[..., None, None]
        v = s["v"][of].double() * s["v_scale"][of].double()[..., None, None]
        k = torch.cat(list(k), 1)[:, :length]                         # (kv, rows, hd)
        v = torch.cat(list(v), 2)[:, :, :length].transpose(1, 2)
        p = (length - c + torch.arange(c, device="cuda"))[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = j > p
        if s["window"]:
            hidden |= (p - j >= s["window"]) & (j >= s["sinks"])
        _weigh(s, y, b, c, k, v, hidden)
    return y


def _exact_cross(s):
    y = s["y"].double()
    for b in range(s["n"]):
        length = s["rows"] if s["length"] is None else int(s["length"][b])
        c = s["t"] if s["count"] is None else int(s["count"][b])
        k, v = (x[b, :length].double().transpose(0, 1) for x in (s["k"], s["v"]))
        _weigh(s, y, b, c, k, v, None)
    return y
