"""AdamW from its formulas in 64 bits (numpy), and the 8-bit rounding of the
moments, for one tensor as a flat array of real elements."""
import numpy as np

BLOCK = 256
U = 2.0 ** -24   # half a step of float32


def step(p, g, m, v, t, lr, b1, b2, eps, wd, clip=1.0):
    """(p, m, v, e): the new values and, for each, how far a computation that
    rounds every product and sum to float32 may be from them.

    A rounding is off by U relative.  m: g' (c rounded, product) 2, b1 and its
    product 2, 1 - b1 and its product 2, the sum 1, so at most 5 on either
    term: 5 U (b1 |m| + (1 - b1) |g'|).  v: g'^2 has 2 * 2 + 1 = 5, times
    1 - b2 (rounded) 7, the sum 8; all terms are positive: 8 U v.
    1 - b^t = -expm1(t ln b): ln b and its product with t 2 (an error d of x = t
    ln b is off by at most d of 1 - e^x), expm1f 2 (one unit in the last place):
    4 U.  lr over it: lr 1, the quotient 1: 6 U.  One over its root: half of 4,
    and rsqrtf 4 (two units): 6 U.
    The denominator: half of v's 8, the root 2 (sqrt.approx.f32 is good to
    2^-23), the constant 6 and its product 1, the sum 1: 14 U.  One over it
    adds 2 (rcp.approx.f32 is good to 2^-23), its product with m 1, the rate 6
    and its product 1: 24 U of the update beside m's own.  p: decay and its
    product 2, the difference 1 on either side: 3 U |p| + (24 + 1 + 5) U
    update(|m| terms).  Second orders are below a tenth of U: every count is
    raised by one.  (The root is that of v + 2^-126: below 1e-11 of eps.)"""
    g = g * clip
    m1 = b1 * m + (1 - b1) * g
    mabs = b1 * np.abs(m) + (1 - b1) * np.abs(g)
    v1 = b2 * v + (1 - b2) * g * g
    rate = lr / (1 - b1 ** t)
    d = np.sqrt(v1) / np.sqrt(1 - b2 ** t) + eps
    p1 = p * (1 - lr * wd) - rate * m1 / d
    # the smallest values are rounded to multiples of 2^-149 instead
    tiny = 2.0 ** -148
    return p1, m1, v1, (U * (4 * np.abs(p) + 31 * rate * mabs / d) + tiny, 6 * U * mabs + tiny,
                        9 * U * v1 + tiny)


def _mix(x):
    x = np.asarray(x, np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def noise(seed, t, ordinal, n, start=0):
    """32 random bits for every element from number `start` on"""
    w = np.uint64(0xffffffff)
    add = lambda a, b: np.uint32((np.uint64(a) + np.uint64(b)) & w)  # noqa: E731
    key = _mix(add(_mix(add(_mix(np.uint32(seed)), t)), ordinal))
    i = np.arange(start, start + n, dtype=np.uint64)
    key = _mix(((np.uint64(key) + (i >> np.uint64(32))) & w).astype(np.uint32))
    return _mix((i & w).astype(np.uint32) ^ key)


def scales(x, top):
    """2^k per block: the least with max finite |x| <= top * 2^k, k >= -126"""
    n = x.size
    y = np.zeros(-(-n // BLOCK) * BLOCK)
    y[:n] = np.where(np.isfinite(x), np.abs(x), 0)
    y = y.reshape(-1, BLOCK).max(1)
    f, e = np.frexp(y / top)              # y / top = f 2^e, 1/2 <= f < 1
    k = np.where(f == 0.5, e - 1, e)
    return np.exp2(np.maximum(np.where(y > 0, k, -126), -126).astype(np.float64))


def spread(s, n):
    return np.repeat(s, BLOCK)[:n]


def round_m(x, s, h):
    """e4m3 values (times the scale) of m; the noise goes below the last of
    three bits; under 2^-6 nothing is left"""
    y = np.abs(x) / spread(s, x.size)
    e = np.frexp(y)[1] - 1
    step_ = np.exp2((e - 3).astype(np.float64))
    u = ((h & np.uint32(0xffff)).astype(np.float64) * 16 + 8) / 2 ** 20
    z = np.floor(y / step_ + u) * step_
    z = np.where(z < 2.0 ** -6, 0, np.minimum(z, np.where(spread(s, x.size) == 2.0 ** 120, 240, 448)))
    return np.copysign(z, x) * spread(s, x.size)


def round_v(x, s, h):
    """e5m2 values (times the scale) of v >= 0; 2^-14 at least where v > 0"""
    y = x / spread(s, x.size)
    e = np.frexp(y)[1] - 1
    step_ = np.exp2((e - 2).astype(np.float64))
    u = ((h >> np.uint32(16)).astype(np.float64) * 32 + 16) / 2 ** 21
    z = np.floor(y / step_ + u) * step_
    z = np.minimum(z, np.where(spread(s, x.size) == 2.0 ** 113, 28672, 57344))
    return np.where(y > 0, np.maximum(z, 2.0 ** -14), 0) * spread(s, x.size)
