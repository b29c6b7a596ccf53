"""The paged KV cache's operators from their definitions, on the CPU: tables with
lists, codes step by step in float32, values in float64."""
import numpy as np
import torch

F = np.float32


class Pages:
    """Tables and the stack of free pages, request by request."""

    def __init__(self, n, most, pages, order=None):
        self.rows = [[] for _ in range(n)]
        self.most, self.pages = most, pages
        self.stack = list(range(pages) if order is None else order)

    def fit(self, lengths, page):
        """False, and nothing done, where the step cannot be made."""
        need = [-(-x // page) for x in lengths]
        if min(lengths) < 0 or max(need) > self.most:
            return False
        back = sum(max(len(r) - k, 0) for r, k in zip(self.rows, need))
        if sum(max(k - len(r), 0) for r, k in zip(self.rows, need)) > len(self.stack) + back:
            return False
        for r, k in reversed(list(zip(self.rows, need))):
            while len(r) > k:
                self.stack.append(r.pop())
        for r, k in zip(self.rows, need):
            while len(r) < k:
                r.append(self.stack.pop())
        return True

    def table(self):
        return torch.tensor([r + [-1] * (self.most - len(r)) for r in self.rows], dtype=torch.int32)

    def held(self):
        return torch.tensor([len(r) for r in self.rows], dtype=torch.int32)

    def free(self):
        return torch.tensor(self.stack + [-7] * (self.pages - len(self.stack)), dtype=torch.int32)

    def left(self):
        return torch.tensor([len(self.stack)], dtype=torch.int32)


class Pool:
    """One half, K's or V's, of a pool: codes (pages, kv, page, hd) and scales."""

    def __init__(self, codes, scale):
        self.codes, self.scale = codes.numpy().astype(np.int8), scale.numpy().astype(F)
        self.page = codes.shape[2]

    def store(self, x, table, start):
        """Rows x (rows, kv, hd) F32 at start.. of the sequence with this table."""
        x, page = x.numpy(), self.page
        for i in range(start // page, (start + len(x) - 1) // page + 1 if len(x) else 0):
            r0, r1 = max(start - i * page, 0), min(start + len(x) - i * page, page)
            rows = x[i * page + r0 - start:i * page + r1 - start]
            at = int(table[i])
            for h in range(x.shape[1]):
                new, was = rows[:, h], self.scale[at, h]
                ok = np.isfinite(new).all() and (r0 == 0 or was >= 0 and np.isfinite(was))
                if not ok:
                    self.scale[at, h] = F(np.nan)
                    self.codes[at, h, r0:r1] = 0
                    continue
                d = np.abs(new).max() * (F(1) / F(127))
                if r0 > 0 and not d > was:
                    d = was
                elif r0 > 0:
                    c = self.codes[at, h, :r0].astype(F) * (was / d)
                    self.codes[at, h, :r0] = np.rint(c).astype(np.int8)
                self.scale[at, h] = d
                with np.errstate(all="ignore"):
                    q = np.rint(new / d) if d > 0 else np.zeros_like(new)
                self.codes[at, h, r0:r1] = np.clip(q, -127, 127).astype(np.int8)

    def values(self):
        """(pages, kv, page, hd) F32."""
        with np.errstate(invalid="ignore"):
            d = np.where((self.scale >= 0) & np.isfinite(self.scale), self.scale, F(np.nan))
            return torch.from_numpy(self.codes.astype(F) * d[:, :, None, None])

    def rows(self, table, length):
        """The rows of one sequence, (length, kv, hd) F32; NaN of a page outside the pool."""
        v = self.values()
        out = torch.full((length, v.shape[1], v.shape[3]), float("nan"))
        for i in range(-(-length // self.page)):
            at, n = int(table[i]), min(self.page, length - i * self.page)
            if 0 <= at < v.shape[0]:
                out[i * self.page:i * self.page + n] = v[at, :, :n].transpose(0, 1)
        return out


def slots(table, length, count, page, t):
    out = torch.full((len(length), t), -1, dtype=torch.int32)
    for b in range(len(length)):
        c = min(max(int(count[b]), 0), t)
        for i in range(c):
            p = int(length[b]) - c + i
            if 0 <= p < table.shape[1] * page and int(table[b, p // page]) >= 0:
                out[b, i] = int(table[b, p // page]) * page + p % page
    return out


EPS = 2.0 ** -24  # half a step of f32


def attend(q, k, v, table, length, count, scale, window=0, sinks=0):
    """(y, bound) in float64 for q (N, T, H, hd) and the pool halves k and v. y is
    NaN where a query sees a block without a finite scale >= 0, a page outside the
    pool, or is not finite itself; bound is NaN where no query is (t >= count).

    How far a result may be, row by row, so that none hides what it does to others:
    a score s_j = scale q.c_j d_j is off by e_j, of hd products summed in f32,
    operands and the scales' products by half steps each (20 more), the difference
    s_j - max and its rounding (2 (|s_j| + |max|)), and q's two F16 pieces, 2^-38 of its
    largest value each: hd max|q| max|k_j|. A weight w_j then moves by w_j (e^(e_j)
    - 1) and their sum by the sum of these; to this come n + 32 half steps of the sum and
    of the weights' own roundings. Pieces hold weight times scale to 2^-39 of 2^14
    times the largest such product, of which half a step is lost twice: 2^-38
    max_i(w_i d_i) |c_j| each; a weight below 2^-126 of the largest may be 0, and a
    result below 2^-126 too."""
    n, t, heads, hd = q.shape
    y = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.full(q.shape, float("nan"), dtype=torch.float64)
    kv, page = k.codes.shape[1], k.page
    group = heads // kv
    for b in range(n):
        ln = min(max(int(length[b]), 0), table.shape[1] * page)
        c = min(max(int(count[b]), 0), t)
        if c == 0:
            continue
        if ln == 0:
            bound[b, :c] = 0.0
            continue
        of = table[b, :-(-ln // page)].long()
        inside = (of >= 0) & (of < len(k.codes))
        of = torch.where(inside, of, 0)

        def rows(pool):  # codes (heads, ln, hd), scales (heads, ln), NaN where there is none
            codes = torch.from_numpy(pool.codes)[of].double().transpose(0, 1).flatten(1, 2)[:, :ln]
            d = torch.from_numpy(pool.scale)[of].double()
            d = torch.where((d >= 0) & (d < float("inf")) & inside[:, None], d, float("nan"))
            d = d.repeat_interleave(page, 0)[:ln].T
            return codes.repeat_interleave(group, 0), d.repeat_interleave(group, 0)

        (kc, kd), (vc, vd) = rows(k), rows(v)
        at = ln - c + torch.arange(c)
        j = torch.arange(ln)
        hidden = j > at[:, None]
        if window:
            hidden |= (j <= at[:, None] - window) & (j >= sinks)
        x = q[b, :c].double().transpose(0, 1)                                  # (heads, c, hd)
        none = torch.isnan(kd + vd)
        lost = (~hidden & none[:, None]).any(-1) | (~torch.isfinite(x).all(-1) & (~hidden).any(-1))
        x = torch.where(torch.isfinite(x), x, 0.0)
        kd, vd = torch.where(none, 0.0, kd), torch.where(none, 0.0, vd)
        kk, vv = kc * kd[..., None], vc * vd[..., None]
        s = (scale * (x @ kk.transpose(1, 2))).masked_fill(hidden, -float("inf"))
        top = s.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
        w = (s - top).exp()
        total = w.sum(-1, keepdim=True)
        w = w / total.clamp_min(1e-300)
        size = abs(scale) * (x.abs() @ kk.abs().transpose(1, 2))
        e = (hd + 20) * EPS * size + abs(scale) * hd * 2.0 ** -38 * x.abs().amax(-1)[..., None] * kk.abs().amax(-1)[:, None]
        e = e + 2 * EPS * (s.abs() + top.abs())
        e = torch.where(hidden, 0.0, torch.expm1(e.nan_to_num(posinf=0.0).clamp_max(700.0)))
        moved = w * (e + (w * e).sum(-1, keepdim=True))
        seen = (~hidden).double()
        far = moved @ vv.abs() + (ln + 32) * EPS * (w @ vv.abs())
        far = far + 2.0 ** -38 * (w * vd[:, None]).amax(-1, keepdim=True) * (seen @ vc.abs())
        far = far + 2.0 ** -126 * (1.0 + seen @ vv.abs())
        res = (w @ vv).masked_fill(lost[..., None], float("nan"))
        y[b, :c] = torch.where(hidden.all(1)[None, :, None], 0.0, res).transpose(0, 1)
        bound[b, :c] = far.nan_to_num(0.0).transpose(0, 1)
    return y, bound
