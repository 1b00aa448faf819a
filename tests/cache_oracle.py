"""The cache operators in numpy, a token and a head at a time, in 64 bits: what the tests hold the kernels to."""
import numpy as np


class Cache:
    """Codes and scales of K or of V: int8 [pages, heads, page, dim], float32 [pages, heads]."""

    def __init__(self, codes, scales):
        self.codes, self.scales = codes, scales
        self.pages, self.heads, self.page, self.dim = codes.shape

    def values(self, table, first, count):
        """Tokens first .. first + count - 1 as float64 [count, heads, dim]; table: the sequence's pages."""
        out = np.zeros((count, self.heads, self.dim))
        for i in range(count):
            p, at = table[(first + i) // self.page], (first + i) % self.page
            out[i] = self.codes[p, :, at].astype(np.float64) * self.scales[p, :, None].astype(np.float64)
        return out

    def write(self, table, first, x):
        """The definition of a write, block by block; x: [count, heads, dim] (float32 values)."""
        done = 0
        while done < len(x):
            p, at = table[(first + done) // self.page], (first + done) % self.page
            n = min(self.page - at, len(x) - done)
            for h in range(self.heads):
                v = x[done:done + n, h].astype(np.float32)
                finite = np.isfinite(v)
                top = np.max(np.abs(np.where(finite, v, 0))).astype(np.float32)
                had = self.scales[p, h] if at else np.float32(0)
                need = np.float32(top * np.float32(1 / 127))
                scale = had if need <= had else max(need, np.float32(had * np.float32(1.25)))
                if scale != had and at and had > 0:
                    old = self.codes[p, h, :at].astype(np.float64)
                    self.codes[p, h, :at] = np.rint(old * float(had) / float(scale)).astype(np.int8)
                if scale == 0:
                    new = np.zeros(v.shape)
                else:
                    new = np.rint(np.where(finite, v, 0).astype(np.float64) / float(scale))
                    new = np.where(np.isposinf(v), 127, np.where(np.isneginf(v), -127, new))
                self.codes[p, h, at:at + n] = new.astype(np.int8)
                self.scales[p, h] = scale
            done += n


def attend(q, k, v, scale, causal=True, window=0):
    """q [n, heads, dim], k and v [tokens, kv heads, dim], all float64 -> out, lse, and what the tolerances are made of:
    sum p |v|, and the largest scale * sum |q| |k| of a row."""
    n, heads, dim = q.shape
    length, kv = k.shape[:2]
    group = heads // kv
    out, lse = np.zeros(q.shape), np.full((n, heads), -np.inf)
    weight, size = np.zeros(q.shape), np.zeros((n, heads))
    token = np.arange(length)
    for i in range(n):
        place = length - n + i
        seen = token <= place if causal else token >= 0
        if window:
            seen &= token > place - window
        if not seen.any():
            continue
        for h in range(heads):
            kk, vv = k[seen, h // group], v[seen, h // group]
            s = kk @ q[i, h] * scale
            top = s.max()
            e = np.exp(s - top)
            lse[i, h] = top + np.log(e.sum())
            p = e / e.sum()
            out[i, h], weight[i, h] = p @ vv, p @ np.abs(vv)
            size[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
    return out, lse, weight, size
