"""The KV cache's operators from their definitions, on the CPU: the block
formats' quantisers step by step in float32, everything else in float64."""
import numpy as np
import torch

BLOCK = 32
UNIT = {"f32": 4, "f16": 2, "bf16": 2, "q8_0": 34, "q4_0": 18}
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = tuple(UNIT)
EPS = 2.0 ** -24  # half a step of f32


def pack(x, kind):
    """F32 values (..., hd) as a cache of `kind` holds them (uint8 blocks, or the
    16- and 32-bit tensor itself)."""
    if kind in FLOAT:
        return x.to(FLOAT[kind])
    f = np.float32
    b = x.numpy().reshape(-1, BLOCK)
    bad = ~np.isfinite(b).all(1)
    b = np.where(bad[:, None], f(0), b)
    rows = np.arange(len(b))
    top = np.abs(b).max(1)
    if kind == "q8_0":
        d = top / f(127)
    else:
        d = b[rows, np.abs(b).argmax(1)] / f(-8)   # numpy's argmax: the first of equals
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(np.abs(d) >= f(2.0 ** -126), f(1) / d, f(0))
        v = b * inv[:, None]
        if kind == "q8_0":
            whole = np.trunc(v)
            q = whole + np.where(np.abs(v - whole) >= f(0.5), np.sign(v), f(0))
            q = q.astype(np.int8).view(np.uint8)
        else:
            q = np.minimum(np.trunc(v + f(8.5)), f(15)).astype(np.uint8)
            q = q[:, :16] | (q[:, 16:] << 4)
        d16 = np.where(bad, np.float16(np.nan), d.astype(np.float16)).astype(np.float16)
    out = np.concatenate([d16.view(np.uint8).reshape(-1, 2), q], 1)
    return torch.from_numpy(out.reshape(*x.shape[:-1], -1).copy())


def values(c, kind):
    """The F32 values that a cache tensor stands for (CPU)."""
    if kind in FLOAT:
        return c.float()
    b = c.numpy().reshape(-1, UNIT[kind])
    d = np.ascontiguousarray(b[:, :2]).view(np.float16).astype(np.float32)
    if kind == "q8_0":
        q = np.ascontiguousarray(b[:, 2:]).view(np.int8).astype(np.float32)
    else:
        q = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float32) - np.float32(8)
    with np.errstate(invalid="ignore", over="ignore"):
        v = q * d
    return torch.from_numpy(v.reshape(*c.shape[:-1], -1))


def handle(S, c, kind, hd):
    """A cache tensor as the binding takes it."""
    return c if kind in FLOAT else (S.Q8Tensor if kind == "q8_0" else S.Q4Tensor)(c, hd)


def attend(q, k, v, length, count, scale, window=0, sinks=0):
    """(y, bound) in float64: q (N, T, H, hd), k, v (N, cap, KV, hd) values; y is
    NaN where no query is (t >= count). bound is how far an F32 result may be: the
    scores' error E (products of hd terms summed in f32, each operand off by a few
    half steps) moves each weight by a factor e^(2E) at most, and the weighted
    sum of n terms adds n more half steps, with 32 for the weights' own roundings
    and the joins of parts. Where f32 ends: a weight e^(s - max) below 2^-126 may
    become 0, which moves a result by at most 2^-126 |v| (the weights' sum is at
    least 1), and a result below 2^-126 may become 0 itself. Where weights go
    through the matrix units as two F16 pieces, 2^15 e^(s - max) = hi + lo, the
    pieces' smallest step is 2^-24: half of it, 2^-25 / 2^15 = 2^-40, is how far a
    weight may be off however small it is, which moves a result by 2^-40 |v|."""
    n, t, heads, hd = q.shape
    group = heads // k.shape[2]
    q = q.double()
    y = torch.full(q.shape, float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(y)
    for b in range(n):
        ln, c = int(length[b]), int(count[b])
        for i in range(c):
            p = ln - c + i
            seen = [j for j in range(max(0, p + 1)) if not window or j > p - window or j < sinks]
            if not seen:
                y[b, i] = 0.0
                continue
            kk, vv = k[b, seen].double(), v[b, seen].double()
            for h in range(heads):
                kh, vh = kk[:, h // group], vv[:, h // group]
                s = scale * (kh @ q[b, i, h])
                w = torch.softmax(s, 0)
                y[b, i, h] = w @ vh
                e = (hd + 16) * EPS * float((kh.abs() @ q[b, i, h].abs()).max()) * abs(scale)
                bound[b, i, h] = (np.expm1(2 * e) + (len(seen) + 32) * EPS) * (w @ vh.abs()) + 2.0 ** -40 * vh.abs().sum(0) + 2.0 ** -126
    return y, bound


def attend_by_row(q, k, v, kind, length, count, scale, window=0, sinks=0):
    """(y, bound) as attend() gives them, with a bound that lets each row of the
    cache err by what is its own alone, so that a row whose weight is nothing, or
    that a query does not see, cannot hide what it does to the others.

    A score s_j = scale q.k_j is off by e_j: hd products summed in f32, operands,
    lo x lo and the scale's product off by half steps each (16 more), the
    difference s_j - max rounded (|s_j| + |max|), and, where operands are two F16
    pieces, 2^-38 of q's largest value for each of q and, f32, 2^-25 of its largest
    for each value of the row k_j: 2^-25 and 2^-38 of hd max|q| max|k_j|. A weight
    then moves by w_j (e^(e_j) - 1), and the sum of weights by E = sum_j w_j (e^(e_j)
    - 1).
    To this come attend()'s n + 32 half steps of the sum and of the joins, and
    2^-126 where f32 ends. Pieces hold a weight to 2^-40 of the largest, which moves a
    result by 2^-40 |v_j| w_max; over f32, times its row's largest value, to 2^-39
    of 2^15 times the largest such product, and V to 2^-25 of its row's largest.
    bf16 has neither: its pieces hold all 24 bits."""
    n, t, heads, hd = q.shape
    group = heads // k.shape[2]
    y = torch.full(q.shape, float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(y)
    for b in range(n):
        ln, c = int(length[b]), int(count[b])
        if ln == 0:
            y[b, :c], bound[b, :c] = 0.0, 2.0 ** -126
        if c == 0 or ln == 0:
            continue
        kk = k[b, :ln].double().repeat_interleave(group, 1).transpose(0, 1)    # (heads, ln, hd)
        vv = v[b, :ln].double().repeat_interleave(group, 1).transpose(0, 1)
        at = ln - c + torch.arange(c)
        j = torch.arange(ln)
        hidden = j > at[:, None]
        if window:
            hidden |= (j <= at[:, None] - window) & (j >= sinks)
        some = ~hidden.all(1)
        # what no query of the sequence sees may be anything at all
        kk, vv = (torch.where(hidden.all(0)[None, :, None], 0.0, x) for x in (kk, vv))
        x = q[b, :c].double().transpose(0, 1)                                  # (heads, c, hd)
        s = scale * (x @ kk.transpose(1, 2))
        s = s.masked_fill(hidden, -float("inf"))
        top = s.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
        w = (s - top).exp()
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
        size = abs(scale) * (x.abs() @ kk.abs().transpose(1, 2))
        kmax, vmax = kk.abs().amax(-1), vv.abs().amax(-1)                      # (heads, ln)
        rows = 2.0 ** -25 if kind == "f32" else 0.0
        e = (hd + 16) * EPS * size + abs(scale) * hd * (rows + 2.0 ** -38) * x.abs().amax(-1)[..., None] * kmax[:, None]
        e = e + EPS * (s.abs() + top.abs())
        e = torch.where(hidden, 0.0, torch.expm1(e.nan_to_num(posinf=0.0).clamp_max(700.0)))
        moved = w * (e + (w * e).sum(-1, keepdim=True))
        far = moved @ vv.abs() + (ln + 32) * EPS * (w @ vv.abs())
        far = far + rows * (w @ vmax[..., None])
        if kind == "f32":
            far = far + ln * 2.0 ** -24 * (w * vmax[:, None]).amax(-1, keepdim=True)
        elif kind != "bf16":
            far = far + 2.0 ** -40 * w.amax(-1, keepdim=True) * ((~hidden).double() @ vv.abs())
        y[b, :c] = torch.where(some[None, :, None], w @ vv, 0.0).transpose(0, 1)
        bound[b, :c] = (far + 2.0 ** -126).transpose(0, 1)
    return y, bound
