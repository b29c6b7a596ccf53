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
                d = np.abs(new).max() / F(127)
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
