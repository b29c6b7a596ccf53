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
