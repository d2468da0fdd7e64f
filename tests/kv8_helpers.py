"""Plain restatements of the 8-bit paged KV cache for its tests: float32 numpy
for what must match bit for bit, float64 for attention."""
from __future__ import annotations

import numpy as np

BLOCK = 16
QMAX = {"int8": 127.0, "e4m3": 448.0}


def _e4m3_table() -> np.ndarray:
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    mag = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    mag[(b & 127) == 127] = np.nan
    return np.where(b & 128, -mag, mag).astype(np.float32)


E4M3 = _e4m3_table()


def decode(codes: np.ndarray, fmt: str) -> np.ndarray:
    return codes.view(np.int8).astype(np.float32) if fmt == "int8" else E4M3[codes]


def encode(x: np.ndarray, fmt: str) -> np.ndarray:
    """Nearest code of float32 values, ties to even, saturating; NaN gives 0."""
    x = np.where(np.isnan(x), np.float32(0), x)
    x = np.clip(x, -QMAX[fmt], QMAX[fmt])
    if fmt == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    mag = np.abs(x).astype(np.float64)
    step = 2.0 ** (np.floor(np.log2(np.maximum(mag, 2.0 ** -6))) - 3)
    q = np.minimum(np.rint(mag / step) * step, 448.0)
    code = np.searchsorted(E4M3[:127].astype(np.float64), q)  # the values of codes 0 .. 126 rise
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_for(a, fmt: str) -> np.float32:
    """The least power of two s in [2^-64, 2^63] with a <= qmax * s."""
    s = 2.0 ** -64
    while s < 2.0 ** 63 and float(a) > QMAX[fmt] * s:
        s *= 2
    return np.float32(s)


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, pos, layout: str, inverse=False) -> np.ndarray:
    """float32, each product and sum rounded on its own; x [tokens, heads, D]."""
    x = x.astype(np.float32)
    half = cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    if inverse:
        s = -s
    out = x.copy()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    return out


class Pool:
    """One layer's pool on the host."""

    def __init__(self, pages, kv_heads, page, dim, fmt, rng, fill="random"):
        self.shape, self.fmt, self.page, self.dim = (pages, kv_heads, page, dim), fmt, page, dim
        self.k, self.v = (self._codes(rng) for _ in range(2))
        blocks = (pages, kv_heads, page // BLOCK)
        self.ks, self.vs = ((2.0 ** rng.integers(-8, -4, blocks)).astype(np.float32) for _ in range(2))

    def _codes(self, rng):
        if self.fmt == "int8":
            return rng.integers(-127, 128, self.shape).astype(np.int8).view(np.uint8)
        c = rng.integers(0, 256, self.shape).astype(np.uint8)
        return np.where((c & 127) > 0x70, c & 0xF0, c).astype(np.uint8)  # magnitudes up to 240, no NaN

    def rows(self, which, row, n) -> np.ndarray:
        """[kv_heads, n, D] float64: the first n tokens of the table row."""
        codes, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        ids = row[:-(-n // self.page)]
        x = decode(codes[ids], self.fmt).astype(np.float64)
        x *= np.repeat(scale[ids].astype(np.float64), BLOCK, axis=2)[..., None]
        return x.transpose(1, 0, 2, 3).reshape(self.shape[1], -1, self.dim)[:, :n]

    def append(self, which, row, start, x: np.ndarray):
        """x [n, kv_heads, D] float32 at positions start .. start + n - 1."""
        codes, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        n = x.shape[0]
        for blk in range(start // BLOCK, (start + n + BLOCK - 1) // BLOCK if n else 0):
            p0 = blk * BLOCK
            lo, hi = max(start - p0, 0), min(start + n - p0, BLOCK)
            page, at = row[p0 // self.page], p0 % self.page
            for h in range(self.shape[1]):
                new = x[p0 + lo - start:p0 + hi - start, h]
                fin = np.abs(new[np.isfinite(new)])
                s = scale_for(fin.max() if fin.size else 0.0, self.fmt)
                cell = codes[page, h, at:at + BLOCK]
                if lo > 0:
                    old = scale[page, h, at // BLOCK]
                    s = max(s, old)
                    if s > old:
                        cell[:lo] = encode(decode(cell[:lo], self.fmt) * np.float32(old / s), self.fmt)
                cell[lo:hi] = encode(new * np.float32(1.0 / s), self.fmt)
                scale[page, h, at // BLOCK] = s


def attention(q, pool: Pool, rows, lens, cu, scale, causal=True, window=0):
    """float64 output of q [tokens, heads, D]; sum_j max(p_j, f) |v_j|, f such
    that 1e-5 f is 2^-39 of the row's largest p (a float16 operand that holds
    it as 2^14 ends at 2^-25: smaller p are no longer told apart); and the size
    of the sums behind each row's scores, max_j scale sum_d |q_d k_jd|."""
    T, H, D = q.shape
    g = H // pool.shape[1]
    out, bound, size = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H, 1))
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = pool.rows("k", rows[b], n), pool.rows("v", rows[b], n)
        m = cu[b + 1] - cu[b]
        p = np.arange(n - m, n)[:, None]
        j = np.arange(n)[None]
        seen = (j <= p) if causal else np.ones((m, n), bool)
        if window:
            seen &= j > p - window
        for h in range(H):
            s = np.where(seen, (q[cu[b]:cu[b + 1], h].astype(np.float64) @ k[h // g].T) * scale, -np.inf)
            mx = s.max(axis=1, keepdims=True)
            e = np.where(seen, np.exp(s - np.where(np.isfinite(mx), mx, 0.0)), 0.0)
            tot = e.sum(axis=1, keepdims=True)
            e = e / np.where(tot > 0, tot, 1.0)
            out[cu[b]:cu[b + 1], h] = e @ v[h // g]
            least = 2.0 ** -39 / 1e-5 * e.max(axis=1, keepdims=True)
            bound[cu[b]:cu[b + 1], h] = np.where(seen, np.maximum(e, least), 0.0) @ np.abs(v[h // g])
            a = (np.abs(q[cu[b]:cu[b + 1], h]).astype(np.float64) @ np.abs(k[h // g]).T) * scale
            size[cu[b]:cu[b + 1], h, 0] = np.where(seen, a, 0.0).max(axis=1, initial=0.0)
    return out, bound, size


def table_for(rng, lens, page, pages, spare=1):
    """A table of shuffled pages for sequences of these lengths."""
    order = rng.permutation(pages)
    cap = max(-(-n // page) for n in lens) + spare
    table = np.full((len(lens), cap), -1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    return table


# How far outputs may be from float64.  A float32 score is off by up to 2^-21
# of the sum of its terms' magnitudes (2^-22 from q's two 11-bit parts, as much
# from the float32 sums, the scaling and the exponent's argument), which moves
# every probability, and their sum, by that much; 1e-5 covers the rest in
# float32.  16-bit outputs add half a unit of the output's rounding (8 and 11
# significant bits) and the probabilities' rounding to 11 bits.
def attention_tolerance(dtype: str, out, bound, size):
    tol = (1e-5 + 2 * 2.0 ** -21 * size) * bound
    if dtype == "f32":
        return tol
    unit, tiny = (2.0 ** -8, 0.0) if dtype == "bf16" else (2.0 ** -11, 2.0 ** -25)
    return unit * 1.001 * np.abs(out) + tol + 2.0 ** -11 * 1.01 * bound + tiny
