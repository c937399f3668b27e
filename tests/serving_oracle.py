"""The serving operators' definitions in numpy float64, the oracle of tests/test_serving_*.py."""
import numpy as np

E4M3_MAX = 448.0


def bf16(x):
    """Float32 values rounded to BF16 (nearest even), as Float32."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)


def e4m3_values():
    """The value of each E4M3 byte."""
    out = np.empty(256)
    for i in range(256):
        e, m = (i >> 3) & 15, i & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[i] = np.nan if i & 127 == 127 else (-v if i & 128 else v)
    return out


E4M3 = e4m3_values()


def quantise(x):
    """E4M3 bytes and scale bytes of rows (..., width): the smallest power of two (>= 2^-126) that brings the largest
    finite magnitude to 448 or below, values to the nearest (ties to the even code), nonfinite to NaN."""
    x = np.asarray(x, np.float32).astype(np.float64)
    top = np.where(np.isfinite(x), np.abs(x), 0).max(-1)
    e = np.zeros(top.shape, np.int64)
    for i in np.ndindex(top.shape):
        if top[i] > 0:
            k = -126
            k = max(k, int(np.floor(np.log2(top[i]))) - 10)
            while np.ldexp(E4M3_MAX, k) < top[i]:
                k += 1
            e[i] = k
    y = x * np.ldexp(1.0, -e)[..., None]
    grid = E4M3[:127]
    mag = np.abs(np.where(np.isfinite(y), y, 0))
    hi = np.clip(np.searchsorted(grid, mag), 0, 126)
    lo = np.clip(hi - 1, 0, 126)
    dl, dh = mag - grid[lo], grid[hi] - mag
    code = np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    code = np.where(mag == grid[hi], hi, code) | np.where(np.signbit(y), 128, 0)
    return np.where(np.isfinite(y), code, 127).astype(np.uint8), (e + 127).astype(np.uint8)


def norm_rope(x, weight, positions, eps, theta):
    """(rows, heads, width) float64."""
    x = np.asarray(x, np.float64)
    width = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    a = np.asarray(positions, np.float64)[:, None] * theta ** (-2.0 * np.arange(width // 2) / width)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    u, v = x[..., :width // 2], x[..., width // 2:]
    return np.concatenate((u * c - v * s, v * c + u * s), -1)


def attend(q, keys, values):
    """One request: q (heads, width), keys / values (kv_heads, n, width), float64.  Returns y and, per element, the
    sum of p |v| and the largest sum |q k| / sqrt(width) over the keys (the scales of the rounding bounds)."""
    heads, width = q.shape
    kv, n = keys.shape[:2]
    q = np.asarray(q, np.float64).reshape(kv, heads // kv, width)
    if n == 0:
        z = np.zeros((heads, width))
        return z, z, np.zeros((heads, 1))
    s = np.einsum("hgd,hnd->hgn", q, keys) / np.sqrt(width)
    mass = np.einsum("hgd,hnd->hgn", np.abs(q), np.abs(keys)).max(-1) / np.sqrt(width)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    y = np.einsum("hgn,hnd->hgd", p, values)
    w = np.einsum("hgn,hnd->hgd", p, np.abs(values))
    return y.reshape(heads, width), w.reshape(heads, width), mass.reshape(heads, 1)


class PagedCacheOracle:
    """A paged cache on the host: payloads as the device holds them, and the values they stand for."""

    def __init__(self, rng, pages, kv_heads, page_size, width, dtype):
        self.dtype, self.page_size = dtype, page_size
        shape = (pages, kv_heads, page_size, width)
        self.raw, self.scales = [], []
        for _ in range(2):
            x = rng.standard_normal(shape).astype(np.float32)
            raw, scale = self.encode(x)
            self.raw.append(raw)
            self.scales.append(scale)

    def encode(self, x):
        if self.dtype == "F32":
            return np.array(x, np.float32), None
        if self.dtype == "BF16":
            return (bf16(x).view(np.uint32) >> 16).astype(np.uint16), None
        if self.dtype == "F16":
            with np.errstate(over="ignore"):
                return np.asarray(x, np.float32).astype(np.float16).view(np.uint16), None
        return quantise(x)

    def values(self, side):
        raw = self.raw[side]
        if self.dtype == "F32":
            return raw.astype(np.float64)
        if self.dtype == "BF16":
            return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        if self.dtype == "F16":
            return raw.view(np.float16).astype(np.float64)
        return E4M3[raw] * np.ldexp(1.0, self.scales[side].astype(np.int64) - 127)[..., None]

    def append(self, side, x, tables, sequences, positions):
        raw, scale = self.encode(x)
        for r in range(len(x)):
            if sequences[r] < 0 or positions[r] < 0:
                continue
            page, slot = tables[sequences[r], positions[r] // self.page_size], positions[r] % self.page_size
            self.raw[side][page, :, slot] = raw[r]
            if scale is not None:
                self.scales[side][page, :, slot] = scale[r]

    def rows(self, side, tables, sequence, n):
        """(kv_heads, n, width) of a request's first n tokens."""
        v = self.values(side)
        if n == 0:
            return np.zeros((v.shape[1], 0, v.shape[3]))
        at = np.arange(n)
        return v[tables[sequence, at // self.page_size], :, at % self.page_size].transpose(1, 0, 2)


def tables_for(rng, lengths, page_size, spare=2):
    """Page tables of requests with these lengths, pages in a random order, unused entries -1; and the page count."""
    blocks = [-(-int(n) // page_size) for n in lengths]
    order = rng.permutation(sum(blocks) + spare).astype(np.int32)
    table = np.full((len(lengths), max(1, max(blocks, default=0))), -1, np.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += b
    return table, sum(blocks) + spare
