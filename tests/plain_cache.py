"""The coefficient cache from its definition in 64 bits (numpy)."""
import numpy as np

RUN = 32   # codes that share a scale


def quantise(x, fmt):
    """x: float32 [..., n], n a multiple of 32 -> (values of the codes, scales),
    float64; a code that stands for no number is NaN"""
    y = x.astype(np.float64).reshape(*x.shape[:-1], -1, RUN)
    fine = np.isfinite(y)
    top = np.where(fine, np.abs(y), 0).max(-1)
    f, e = np.frexp(top / (127.0 if fmt == "int8" else 448.0))
    k = np.where(top > 0, np.where(f == 0.5, e - 1, e), -126)
    s = np.exp2(np.maximum(k, -126).astype(np.float64))
    with np.errstate(invalid="ignore"):
        z = np.where(fine, y, 0) / s[..., None]
    if fmt == "int8":
        c = np.round(z)
    else:
        e = np.frexp(z)[1] - 1
        step = np.exp2(np.maximum(e - 3, -9).astype(np.float64))
        c = np.round(z / step) * step
    # what is read back stays below 2^128
    most = np.where(s == 2.0 ** 122, 63, 127) if fmt == "int8" else np.where(s == 2.0 ** 120, 240, 448)
    c = np.clip(c, -most[..., None], most[..., None])
    return np.where(fine, c, np.nan).reshape(x.shape), s


class Ring:
    """what CoefCache holds, in float64"""

    def __init__(self, rows, capacity, ncoef, fmt):
        self.fmt, self.capacity = fmt, capacity
        self.codes = np.zeros((rows, capacity, 2 * ncoef))
        self.scales = np.full((rows, capacity, ncoef // 16), 2.0 ** -126)
        self.length = np.zeros(rows, np.int64)

    def append(self, heap, counts=None):
        """heap: complex64 [rows, S, ncoef]"""
        x = np.ascontiguousarray(heap).view(np.float32)
        for r in range(x.shape[0]):
            n = x.shape[1] if counts is None else min(max(int(counts[r]), 0), x.shape[1])
            for k in range(n):
                slot = self.length[r] % self.capacity
                self.codes[r, slot], self.scales[r, slot] = quantise(x[r, k], self.fmt)
                self.length[r] += 1

    def window(self, n, end=None):
        """[rows, n, ncoef, 2] float64"""
        rows, _, m = self.codes.shape
        out = np.zeros((rows, n, m))
        for r in range(rows):
            e = self.length[r] if end is None else end[r]
            for j in range(n):
                k = e - n + j
                if max(0, self.length[r] - self.capacity) <= k < self.length[r]:
                    s = k % self.capacity
                    out[r, j] = self.codes[r, s] * np.repeat(self.scales[r, s], RUN)
        return out.reshape(rows, n, m // 2, 2)
