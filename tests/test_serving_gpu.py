"""The operators of a batch of several requests (stb_op_qk_norm_rope, stb_op_paged_append / read / attention,
stb_linear_pool) against their definitions in float64 (tests/serving_oracle.py).

Tolerances, from the arithmetic:
* norm and rotation, y = fma(a, c, -(b s)) with a = x inv w, b = x' inv w': in half steps h of Float32 (2^-24), inv, the two
  products of a and c are rounded once each (4 h |a c|), likewise those of b s and b s itself (5 h |b s|), and the sum
  once (h |y|).  |a c| + |b s| <= sqrt(2) pair, so 5 sqrt(2) < 7.1 h of the pair's magnitude and h |y|; the norm's factor
  before its rounding (2^-43) and the angle (two double roundings at positions below 2^20: 5e-10) add 1e-9 of the pair.
* cache write and read: equal bits.
* attention in Float32: a score's rounding error is at most (width + 8) 2^-24 of its sum |q k| / sqrt(width) (one
  rounding per product and addition, of any order), a weight moves by e^(2 |error|) - 1 of itself against the sum,
  and a sum of n weighted values by at most (n + 16) 2^-23 of the sum of |p v| (truncating additions counted as a
  whole step).  Beside that worst case, roundings of random sign: the 2-norm of the error stays within 32 half
  steps (2e-6) of the output's.
* adapted Linear: the Linear's own 1e-5 (1 + |e|).
"""
import numpy as np
import pytest

import oracle
from scalatorch import ffm
from serving_oracle import E4M3, PagedCacheOracle, attend, bf16, norm_rope, quantise, tables_for

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24
CODES = {"F32": ffm.STB_F32, "BF16": ffm.STB_BF16, "F16": ffm.STB_F16, "E4M3": ffm.STB_E4M3}


class Held:
    """Uploads that are released together."""

    def __init__(self, session):
        self.s, self.kept = session, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for t in reversed(self.kept):
            self.s.release(t)

    def keep(self, t):
        self.kept.append(t)
        return t

    def f32(self, a):
        return self.keep(self.s.upload(np.asarray(a, np.float32)))

    def ints(self, a):
        return self.keep(self.s.upload_ints(a))

    def raw(self, a, dtype):
        t = self.keep(self.s.allocate(a.shape, dtype))
        a = np.ascontiguousarray(a)
        if a.size:
            ffm.call("stb_upload", self.s.handle, a.ctypes.data, a.nbytes, t.address)
        return t

    def cache(self, o):
        data = [self.raw(r, CODES[o.dtype]) for r in o.raw]
        scales = [self.raw(x, ffm.STB_U8) for x in o.scales] if o.dtype == "E4M3" else []
        return self.s.paged_cache(*data, *scales)


def raw_of(session, t, like):
    return session.download_raw(t).view(like.dtype).reshape(like.shape)


# ------------------------------------------------------------------ norm and rotation


def check_norm_rope(got, x, w, pos, eps, theta):
    want = norm_rope(x, w, pos, eps, theta)
    half = want.shape[-1] // 2
    pair = np.hypot(want[..., :half], want[..., half:])
    tol = HALF * np.abs(want) + (7.1 * HALF + 1e-9) * np.concatenate((pair, pair), -1) + 1e-37
    np.testing.assert_array_less(np.abs(got.astype(np.float64) - want), tol)


@pytest.mark.parametrize("rows,heads,kv,width,normed,theta", [
    (1, 9, 3, 64, True, 10000.0), (5, 4, 2, 128, True, 500000.0), (33, 8, 1, 128, False, 10000.0), (3, 2, 2, 2, True, 10000.0),
    (2, 3, 3, 80, True, 1e6), (7, 5, 1, 96, True, 10000.0), (2, 2, 1, 256, True, 10000.0), (2, 1, 1, 512, True, 10000.0),
    (3, 7, 1, 66, True, 0.5), (700, 14, 2, 64, True, 10000.0), (2, 2, 1, 34, True, 1.0), (9, 64, 8, 128, True, 500000.0)])
def test_qk_norm_rope(session, rows, heads, kv, width, normed, theta):
    rng = np.random.default_rng(rows * 31 + width)
    q, k = (rng.standard_normal((rows, n, width)).astype(np.float32) * 3 for n in (heads, kv))
    wq, wk = ((1 + 0.3 * rng.standard_normal(width)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 1 << 20, rows)
    pos[0] = 0
    with Held(session) as h:
        ws = (h.f32(wq), h.f32(wk)) if normed else (None, None)
        yq, yk = session.qk_norm_rope(h.f32(q), h.f32(k), *ws, h.ints(pos), 1e-5, theta)
        h.keep(yq), h.keep(yk)
        check_norm_rope(session.download(yq), q, wq if normed else None, pos, 1e-5, theta)
        check_norm_rope(session.download(yk), k, wk if normed else None, pos, 1e-5, theta)


@pytest.mark.parametrize("width", [64, 36])
def test_qk_norm_rope_of_tiny_and_large_heads(session, width):
    """Heads whose mean square leaves Float32 at either end, and heads of zeros, beside ordinary ones."""
    rng = np.random.default_rng(8)
    rows, eps = 5, 1e-100
    x = rng.standard_normal((rows, 2, width))
    x[0] *= 1e-40
    x[1] *= 1e37
    x[2] = 0.0
    x[3, 0] *= 1e-30
    x[3, 1, :-1] = 0.0
    x[3, 1, -1] = 1e-44
    x = x.astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    pos = np.array([0, 7, 3, 1, 50])
    with Held(session) as h:
        dw, dp = h.f32(w), h.ints(pos)
        q, k = session.qk_norm_rope(h.f32(x), h.f32(x[:, :1]), dw, dw, dp, eps, 1e4)
        h.keep(q), h.keep(k)
        check_norm_rope(session.download(q), x, w, pos, eps, 1e4)
        check_norm_rope(session.download(k), x[:, :1], w, pos, eps, 1e4)


def test_qk_norm_rope_in_the_rows_of_a_fused_projection_and_in_place(session):
    """q and k as columns of one matrix whose rows have an odd length (no 16-byte alignment), one weight only, padding
    rows left as they were; then in place; extreme rows (zeros, huge, tiny, infinite)."""
    rng = np.random.default_rng(5)
    rows, heads, kv, width, lead = 11, 3, 1, 64, 5
    fused = rng.standard_normal((rows, lead + (heads + 2 * kv) * width)).astype(np.float32)
    fused[2, lead:lead + width] = 0
    fused[3, lead:lead + width] *= 1e30
    fused[4, lead:lead + width] *= 1e-30
    pos = np.array([3, -1, 5, 6, 7, 100000, 0, -7, 1, 2, 77])
    w = (1 + 0.3 * rng.standard_normal(width)).astype(np.float32)
    real = pos >= 0
    q0 = fused[:, lead:lead + heads * width].reshape(rows, heads, width)
    k0 = fused[:, lead + heads * width:lead + (heads + kv) * width].reshape(rows, kv, width)
    with Held(session) as h:
        df, dp, dw = h.f32(fused), h.ints(pos), h.f32(w)
        q, k = h.keep(session.columns(df, lead, (heads, width))), h.keep(session.columns(df, lead + heads * width, (kv, width)))
        out = h.keep(session.fill((rows, heads, width), 7.0)), h.keep(session.fill((rows, kv, width), 7.0))
        session.qk_norm_rope(q, k, None, dw, dp, 1e-6, 10000.0, out=out)
        yq, yk = session.download(out[0]), session.download(out[1])
        check_norm_rope(yq[real], q0[real], None, pos[real], 1e-6, 10000.0)
        check_norm_rope(yk[real], k0[real], w, pos[real], 1e-6, 10000.0)
        assert np.all(yq[~real] == 7.0) and np.all(yk[~real] == 7.0)
        session.qk_norm_rope(q, k, dw, dw, dp, 1e-6, 10000.0, out=(q, k))
        got = session.download(df)
        check_norm_rope(got[real, lead:lead + heads * width].reshape(-1, heads, width), q0[real], w, pos[real], 1e-6, 10000.0)
        check_norm_rope(got[real, lead + heads * width:lead + (heads + kv) * width].reshape(-1, kv, width), k0[real], w, pos[real], 1e-6, 10000.0)
        untouched = np.ones(fused.shape, bool)
        untouched[real, lead:lead + (heads + kv) * width] = False
        assert np.array_equal(got[untouched].view(np.uint32), fused[untouched].view(np.uint32))
        bad = fused[:, lead:lead + width].reshape(rows, 1, width).copy()
        bad[0, 0, 3], bad[5, 0, 9] = np.inf, np.nan
        y, z = session.qk_norm_rope(h.f32(bad), h.f32(bad), dw, dw, dp)
        h.keep(y), h.keep(z)
        got = session.download(y)
        assert np.isnan(got[0]).any() and np.isnan(got[5]).any() and np.isfinite(got[[2, 3, 4, 6, 8]]).all()


# ------------------------------------------------------------------ the paged cache


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16", "E4M3"])
@pytest.mark.parametrize("kv,width,page,tokens", [(3, 64, 16, [5, 1, 40]), (1, 20, 1, [3, 2]), (8, 128, 7, [17, 1, 1, 30]),
                                                  (2, 256, 32, [33]), (1, 33, 4, [6, 1]), (2, 512, 16, [3])])
def test_paged_append_and_read(session, dtype, kv, width, page, tokens):
    """Tokens of several requests at offsets inside their pages, with padding rows between them, in caches that already
    hold others': the whole cache's bits afterwards, and the rows back in both layouts."""
    rng = np.random.default_rng(kv * 1000 + width)
    starts = rng.integers(0, 2 * page + 3, len(tokens))
    tables, pages = tables_for(rng, starts + tokens, page)
    o = PagedCacheOracle(rng, pages, kv, page, width, dtype)
    seq = np.concatenate([np.full(n, i) for i, n in enumerate(tokens)] + [[-1, 0, -3]])
    pos = np.concatenate([s + np.arange(n) for s, n in zip(starts, tokens)] + [[4, -1, -2]])
    rows = len(seq)
    x = [(rng.standard_normal((rows, kv, width)) * 10.0 ** rng.integers(-6, 6, (rows, kv, 1))).astype(np.float32) for _ in range(2)]
    x[0][0, 0] = 0.0
    x[1][0, 0, :3] = [448.0, -449.0, 1e-4]
    with Held(session) as h:
        cache = h.cache(o)
        dt, ds, dp = h.ints(tables), h.ints(seq), h.ints(pos)
        cache.append(h.f32(x[0]), h.f32(x[1]), dt, ds, dp)
        for side in range(2):
            o.append(side, x[side], tables, seq, pos)
            assert np.array_equal(raw_of(session, cache.tensors[side], o.raw[side]), o.raw[side])
            if dtype == "E4M3":
                assert np.array_equal(raw_of(session, cache.tensors[2 + side], o.scales[side]), o.scales[side])
        real = (seq >= 0) & (pos >= 0)
        for first in (False, True):
            got = cache.read(dt, ds, dp, heads_first=first)
            for side in range(2):
                v = o.values(side)
                want = np.zeros((rows, kv, width))
                want[real] = v[tables[seq[real], pos[real] // page], :, pos[real] % page]
                y = session.download(h.keep(got[side])).astype(np.float64)
                assert np.array_equal(y.transpose(1, 0, 2) if first else y, want)
        out = h.keep(session.fill((rows, kv, width), 9.0)), h.keep(session.fill((rows, kv, width), 9.0))
        cache.read(dt, ds, dp, out=out)
        assert np.all(session.download(out[0])[~real] == 9.0) and np.all(session.download(out[1])[~real] == 9.0)


def test_paged_append_of_e4m3_borders(session):
    """Every tie and border of the grid, scales at the ends of the range, subnormals, infinities and NaNs."""
    width, page = 512, 4
    grid = E4M3[:127]
    mid = (grid[1:] + grid[:-1]) / 2
    row = np.concatenate((grid, mid, np.nextafter(mid.astype(np.float32), np.float32(1e9)), np.nextafter(mid.astype(np.float32), np.float32(0))))
    row = np.concatenate((row, [0.0] * (width - len(row))))[:width].astype(np.float32)
    rows = [row, -row, row * np.float32(2.0 ** 119), row * np.float32(2.0 ** -140), row * 0, row * np.float32(1.75), row * np.float32(1.7500001)]
    special = row.copy()
    special[[1, 5, 9]] = [np.inf, -np.inf, np.nan]
    tiny = np.zeros(width, np.float32)
    tiny[:3] = [1e-45, -1e-40, 1.1754944e-38]
    top = row * 0
    top[:2] = [3.4028235e38, -1.0]
    x = np.stack(rows + [special, tiny, top])[:, None]
    n = len(x)
    rng = np.random.default_rng(1)
    o = PagedCacheOracle(rng, 4, 1, page, width, "E4M3")
    tables, seq, pos = np.array([[2, 0, 3]]), np.zeros(n, int), np.arange(n)
    with Held(session) as h:
        cache = h.cache(o)
        cache.append(h.f32(x), h.f32(x[::-1].copy()), h.ints(tables), h.ints(seq), h.ints(pos))
        for side, v in ((0, x), (1, x[::-1])):
            o.append(side, v, tables, seq, pos)
            assert np.array_equal(raw_of(session, cache.tensors[2 + side], o.scales[side]), o.scales[side])
            got, want = raw_of(session, cache.tensors[side], o.raw[side]), o.raw[side]
            nan = want & 127 == 127
            assert np.array_equal(got[~nan], want[~nan]) and np.all(got[nan] & 127 == 127)


def test_paged_append_from_columns(session):
    """k and v straight out of a fused projection's rows of odd length."""
    rng = np.random.default_rng(8)
    rows, heads, kv, width, page = 6, 2, 2, 48, 16
    fused = rng.standard_normal((rows, (heads + 2 * kv) * width + 3)).astype(np.float32)
    tables, pages = tables_for(rng, [rows], page)
    for dtype in ("E4M3", "BF16"):
        o = PagedCacheOracle(rng, pages, kv, page, width, dtype)
        seq, pos = np.zeros(rows, int), np.arange(rows)
        with Held(session) as h:
            cache, df = h.cache(o), h.f32(fused)
            at = [heads * width + 1, (heads + kv) * width + 1]
            k, v = (h.keep(session.columns(df, a, (kv, width))) for a in at)
            cache.append(k, v, h.ints(tables), h.ints(seq), h.ints(pos))
            for side in range(2):
                o.append(side, fused[:, at[side]:at[side] + kv * width].reshape(rows, kv, width), tables, seq, pos)
                assert np.array_equal(raw_of(session, cache.tensors[side], o.raw[side]), o.raw[side])


# ------------------------------------------------------------------ attention over the paged cache


def check_attend(session, q, o, tables, lengths, h, cache=None, **kw):
    cache = cache or h.cache(o)
    y = h.keep(cache.attend(h.f32(q), h.ints(tables), h.ints(lengths), **kw))
    got = session.download(y).astype(np.float64)
    wants = []
    for b, n in enumerate(lengths):
        n = max(0, int(n))
        k, v = (o.rows(side, tables, b, n) for side in range(2))
        want, mass, score = attend(q[b], k, v)
        tol = (np.expm1(2 * (q.shape[2] + 8) * HALF * score) + (n + 16) * 2 * HALF) * mass + 1e-37
        np.testing.assert_array_less(np.abs(got[b] - want), tol, err_msg=f"request {b} of length {n}")
        wants.append(want)
    want = np.stack(wants)
    assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want) + 1e-30
    return y


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16", "E4M3"])
@pytest.mark.parametrize("heads,kv,width,page,lengths", [
    (9, 3, 64, 16, [33]), (8, 1, 128, 16, [1, 0, 16, 17, 300]), (4, 4, 128, 8, [15, 129]), (16, 1, 128, 32, [70, 5]),
    (12, 4, 96, 16, [50, 0, 2, 64]), (5, 1, 80, 7, [41, 8]), (16, 2, 256, 64, [130, 1]), (7, 7, 20, 1, [9]), (2, 1, 33, 5, [37]),
    (3, 1, 512, 16, [20, 33]), (40, 2, 64, 16, [260, 31]), (8, 8, 32, 16, [100]), (6, 2, 16, 48, [200, 47, 49])])
def test_paged_attention(session, dtype, heads, kv, width, page, lengths):
    rng = np.random.default_rng(heads * 100 + width)
    tables, pages = tables_for(rng, lengths, page)
    o = PagedCacheOracle(rng, pages, kv, page, width, dtype)
    q = rng.standard_normal((len(lengths), heads, width)).astype(np.float32) * 2
    with Held(session) as h:
        check_attend(session, q, o, tables, lengths, h)


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16", "E4M3"])
@pytest.mark.parametrize("heads,kv,width,page,lengths", [(8, 1, 128, 16, [9001]), (4, 2, 64, 64, [1, 5000, 0, 700, 2049, 31]),
                                                         (6, 2, 96, 24, [3000, 1500])])
def test_paged_attention_split_over_a_long_cache(session, dtype, heads, kv, width, page, lengths):
    rng = np.random.default_rng(width)
    tables, pages = tables_for(rng, lengths, page)
    o = PagedCacheOracle(rng, pages, kv, page, width, dtype)
    q = rng.standard_normal((len(lengths), heads, width)).astype(np.float32)
    with Held(session) as h:
        cache = h.cache(o)
        y = check_attend(session, q, o, tables, lengths, h, cache)
        z = h.keep(cache.attend(h.f32(q), h.ints(tables), h.ints(lengths)))
        assert np.array_equal(session.download(y).view(np.uint32), session.download(z).view(np.uint32))


def test_paged_attention_of_many_requests(session):
    """More requests than SMs, most of them short, some empty; a length per request from 0 to 400."""
    rng = np.random.default_rng(77)
    lengths = rng.integers(0, 40, 500)
    lengths[::50] = rng.integers(100, 400, 10)
    lengths[3:9] = 0
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, 2, 16, 64, "BF16")
    q = rng.standard_normal((500, 8, 64)).astype(np.float32)
    with Held(session) as h:
        check_attend(session, q, o, tables, lengths, h)


@pytest.mark.parametrize("dtype", ["BF16", "E4M3"])
@pytest.mark.parametrize("batch,heads,kv,width,longest", [(1100, 4, 1, 64, 20), (60, 8, 4, 128, 40), (200, 16, 1, 128, 33), (1, 8, 8, 64, 9850),
                                                          (1, 24, 3, 80, 4000), (2, 2, 2, 64, 60), (32, 32, 8, 128, 300), (21, 16, 8, 64, 900), (100, 40, 2, 96, 800)])
def test_paged_attention_by_batch(session, dtype, batch, heads, kv, width, longest):
    """More requests than one launch takes; many that a warp, and longer ones that a block each takes whole; one request whose
    items take whole blocks."""
    rng = np.random.default_rng(batch + width)
    lengths = rng.integers(0, longest + 1, batch)
    lengths[-1] = longest
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, kv, 16, width, dtype)
    q = rng.standard_normal((batch, heads, width)).astype(np.float32)
    with Held(session) as h:
        check_attend(session, q, o, tables, lengths, h)


@pytest.mark.parametrize("dtype", ["F32", "BF16", "E4M3"])
def test_paged_attention_of_tiny_and_large_values(session, dtype):
    """Values near the lowest scale that an E4M3 row takes (2^-126) and up to 2^100: results keep their bits.  Tolerance
    as everywhere, and a step of the smallest Float32."""
    rng = np.random.default_rng(14)
    lengths, width = [150, 9, 600, 40], 64
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, 1, 16, width, dtype)
    q = rng.standard_normal((4, 8, width)).astype(np.float32)
    for b, by in enumerate((2.0 ** -119, 2.0 ** -118, 2.0 ** -119, 2.0 ** 100)):
        n = lengths[b]
        o.append(1, (rng.uniform(1, 2, (n, 1, width)) * by).astype(np.float32), tables, np.full(n, b), np.arange(n))
    with Held(session) as h:
        y = session.download(h.keep(h.cache(o).attend(h.f32(q), h.ints(tables), h.ints(lengths)))).astype(np.float64)
        for b, n in enumerate(lengths):
            want, mass, score = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
            tol = (np.expm1(2 * (width + 8) * HALF * score) + (n + 16) * 2 * HALF) * mass + 2.0 ** -149
            np.testing.assert_array_less(np.abs(y[b] - want), tol)


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16", "E4M3"])
def test_paged_attention_of_peaked_and_flat_scores(session, dtype):
    """One key that takes everything, keys far below it, scales that differ by 2^40 between tokens (E4M3), equal keys,
    a request whose scores are all hugely negative."""
    rng = np.random.default_rng(3)
    page, n, width = 16, 150, 128
    tables, pages = tables_for(rng, [n, n, n, 1], page)
    o = PagedCacheOracle(rng, pages, 1, page, width, dtype)
    q = rng.standard_normal((4, 8, width)).astype(np.float32)
    at = np.arange(n)
    k = rng.standard_normal((3 * n, 1, width)).astype(np.float32)
    v = rng.standard_normal((3 * n, 1, width)).astype(np.float32)
    k[70] = q[0, 3] * 4                     # a peak for one head of request 0
    v[:n] *= 2.0 ** rng.integers(-20, 20, (n, 1, 1)) if dtype in ("E4M3", "F32", "BF16") else 1
    k[n:2 * n] = k[n]                       # all keys of request 1 are the same
    k[2 * n:] = -40 * np.sign(q[2, 0]) * np.ones((n, 1, 1), np.float32)
    seq, pos = np.repeat([0, 1, 2], n), np.tile(at, 3)
    for side, x in ((0, k), (1, v)):
        o.append(side, x, tables, seq, pos)
    with Held(session) as h:
        check_attend(session, q, o, tables, [n, n, n, 1], h)


def test_paged_attention_rows_apart_and_tails_untouched(session):
    """Query rows inside a fused projection, outputs inside a wider buffer: nothing else of it changes.  Infinities and
    NaNs behind a request's length (its page's other slots, unused pages) do not reach the result."""
    rng = np.random.default_rng(4)
    heads, kv, width, page, lengths = 4, 2, 64, 16, [21, 5, 0]
    tables, pages = tables_for(rng, lengths, page)
    o = PagedCacheOracle(rng, pages, kv, page, width, "BF16")
    used = np.zeros((pages, page), bool)
    for b, n in enumerate(lengths):
        used[tables[b, np.arange(n) // page], np.arange(n) % page] = True
    for side in range(2):
        poisoned = o.raw[side].transpose(0, 2, 1, 3)
        poisoned[~used] = np.where(rng.random(poisoned[~used].shape) < 0.5, 0x7F80, 0x7FC1)
    fused = rng.standard_normal((3, heads * width + 7)).astype(np.float32)
    with Held(session) as h:
        cache, df = h.cache(o), h.f32(fused)
        wide = h.keep(session.fill((3, heads * width + 9), 5.0))
        q = h.keep(session.columns(df, 3, (heads, width)))
        y = h.keep(session.columns(wide, 4, (heads, width)))
        cache.attend(q, h.ints(tables), h.ints(lengths), out=y)
        got = session.download(wide)
        assert np.all(got[:, :4] == 5.0) and np.all(got[:, 4 + heads * width:] == 5.0)
        want = h.keep(cache.attend(h.f32(fused[:, 3:3 + heads * width].reshape(3, heads, width)), h.ints(tables), h.ints(lengths)))
        part = got[:, 4:4 + heads * width].reshape(3, heads, width)
        assert np.isfinite(part).all() and np.all(part[2] == 0.0)
        np.testing.assert_allclose(part, session.download(want), rtol=0, atol=2e-6)


def test_nan_keys_and_values_inside_a_request_stay_its_own(session):
    rng = np.random.default_rng(6)
    page, lengths = 16, [40, 40, 40]
    tables, pages = tables_for(rng, lengths, page)
    for dtype, nan in (("BF16", 0x7FC0), ("E4M3", 0x7F), ("F16", 0x7E00)):
        o = PagedCacheOracle(rng, pages, 1, page, 64, dtype)
        o.raw[0][tables[0, 1], 0, 3, 5] = nan
        o.raw[1][tables[1, 0], 0, 2, 7] = nan
        q = rng.standard_normal((3, 4, 64)).astype(np.float32)
        with Held(session) as h:
            y = session.download(h.keep(h.cache(o).attend(h.f32(q), h.ints(tables), h.ints(lengths))))
            assert np.isnan(y[0]).all()
            assert np.isnan(y[1, :, 7]).all() and np.isfinite(np.delete(y[1], 7, axis=1)).all()
            assert np.isfinite(y[2]).all()


@pytest.mark.parametrize("page", [-1, -2, -2 ** 31, 4, 2 ** 31 - 1])
def test_attention_reports_any_page_outside_the_cache(session, page):
    rng = np.random.default_rng(10)
    o = PagedCacheOracle(rng, 4, 1, 16, 64, "BF16")
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    tables = np.array([[0, page], [1, 2]])
    with Held(session) as h:
        y = h.keep(h.cache(o).attend(h.f32(q), h.ints(tables), h.ints([20, 20])))
        with pytest.raises(ffm.IllegalStateException, match="paged cache"):
            session.sync()
        got = session.download(y)
        for b, n in ((0, 16), (1, 20)):  # what the bad page held is skipped
            want, _, _ = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
            np.testing.assert_allclose(got[b], want, rtol=0, atol=1e-5)


def test_bad_indices_are_skipped_and_reported(session):
    """Pages outside the cache, positions and lengths behind the table, slots behind the pool: the call names them at the
    next sync, touches nothing else, and the session goes on."""
    rng = np.random.default_rng(9)
    page, width = 16, 64
    o = PagedCacheOracle(rng, 4, 1, page, width, "BF16")
    q = rng.standard_normal((2, 4, width)).astype(np.float32)
    x = rng.standard_normal((3, 1, width)).astype(np.float32)
    with Held(session) as h:
        cache, dq, dx = h.cache(o), h.f32(q), h.f32(x)
        before = [session.download_raw(t) for t in cache.tensors]
        for tables, seq, pos in (([[0, 9]], [0, 0, 0], [16, 17, 31]), ([[0, -1]], [0, 0, 0], [16, 20, 31]),
                                 ([[0, 1]], [0, 0, 0], [32, 33, 2 ** 31 - 1]), ([[0, 1]], [1, 2, 2 ** 31 - 1], [0, 1, 2])):
            dt, ds, dp = h.ints(tables), h.ints(seq), h.ints(pos)
            cache.append(dx, dx, dt, ds, dp)
            with pytest.raises(ffm.IllegalStateException, match="paged cache"):
                session.sync()
            out = h.keep(session.fill((3, 1, width), 3.0)), h.keep(session.fill((3, 1, width), 3.0))
            cache.read(dt, ds, dp, out=out)
            with pytest.raises(ffm.IllegalStateException, match="paged cache"):
                session.sync()
            assert np.all(session.download(out[0]) == 3.0)
        assert all(np.array_equal(session.download_raw(t), b) for t, b in zip(cache.tensors, before))
        for tables, lengths, text in (([[0, 7], [1, 2]], [20, 20], "paged cache"), ([[0, -1], [1, 2]], [17, 20], "paged cache"),
                                      ([[0, 3], [1, 2]], [33, 20], "length"), ([[0, 3], [1, 2]], [2 ** 31 - 1, 20], "length")):
            y = h.keep(cache.attend(dq, h.ints(tables), h.ints(lengths)))
            with pytest.raises(ffm.IllegalStateException, match=text):
                session.sync()
            want, _, _ = attend(q[1], o.rows(0, np.array(tables), 1, 20), o.rows(1, np.array(tables), 1, 20))
            np.testing.assert_allclose(session.download(y)[1], want, rtol=0, atol=1e-5)
        # unused table entries may hold anything; negative lengths are empty rows
        y = h.keep(cache.attend(dq, h.ints([[0, 99], [-5, -5]]), h.ints([16, -4])))
        session.sync()
        assert np.all(session.download(y)[1] == 0.0)


# ------------------------------------------------------------------ adapters of many requests


def pool_case(rng, M, N, K, slots, rank, dtype):
    a = rng.standard_normal((slots, rank, K)).astype(np.float32) / np.sqrt(K)
    b = rng.standard_normal((slots, N, rank)).astype(np.float32) * 0.1
    if dtype == "BF16":
        a, b = bf16(a), bf16(b)
    elif dtype == "F16":
        a, b = (t.astype(np.float16).astype(np.float32) for t in (a, b))
    ranks = rng.integers(1, rank + 1, slots)
    ranks[0] = rank
    return a, b, ranks, rng.uniform(0.5, 2.0, slots).astype(np.float32)


def device_pool(h, a, b, ranks, scales, dtype):
    def up(t):
        if dtype == "F32":
            return h.f32(t)
        bits = (t.view(np.uint32) >> 16).astype(np.uint16) if dtype == "BF16" else t.astype(np.float16).view(np.uint16)
        return h.raw(bits, CODES[dtype])

    return h.s.adapter_pool(up(a), up(b), h.ints(ranks), h.f32(scales))


def adapted(x, w, bias, a, b, ranks, scales, rows):
    y = x.astype(np.float64) @ w.astype(np.float64).T
    for m, t in enumerate(rows):
        if t >= 0:
            r = int(np.clip(ranks[t], 0, a.shape[1]))
            y[m] += scales[t] * (b[t, :, :r].astype(np.float64) @ (a[t, :r].astype(np.float64) @ x[m].astype(np.float64)))
    return y + (0 if bias is None else bias)


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("M,N,K,slots,rank,weight", [
    (1, 64, 64, 1, 1, "BF16"), (1, 1536, 576, 4, 8, "BF16"), (5, 200, 136, 3, 7, "BF16"), (3, 33, 37, 2, 5, "BF16"), (17, 576, 1536, 6, 16, "BF16"),
    (64, 1024, 2048, 9, 33, "BF16"), (70, 512, 1024, 3, 64, "BF16"), (8, 4096, 1024, 8, 64, "BF16"), (9, 256, 512, 4, 12, "F16"), (4, 96, 80, 2, 256, "F32"),
    (130, 384, 640, 70, 8, "BF16"), (40, 4096, 4096, 2, 24, "BF16")])
def test_linear_of_a_pool(session, dtype, M, N, K, slots, rank, weight):
    rng = np.random.default_rng(M * 7 + N)
    x = rng.standard_normal((M, K)).astype(np.float32)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    bias = rng.standard_normal(N).astype(np.float32)
    a, b, ranks, scales = pool_case(rng, M, N, K, slots, rank, dtype)
    rows = rng.integers(-1, slots, M)
    rows[-1] = 0
    with Held(session) as h:
        if weight == "F32":
            dw = h.keep(session.upload_weight_f32(w))
        else:
            bits = oracle.round_bf16(w) if weight == "BF16" else oracle.round_f16(w)
            w = oracle.widen(bits, oracle.BF16 if weight == "BF16" else oracle.F16)
            dw = h.keep(session.upload_weight(bits, CODES[weight]))
        pool = device_pool(h, a, b, ranks, scales, dtype)
        dx, db = h.f32(x), h.f32(bias)
        for choice in (rows, np.full(M, -1), np.full(M, slots - 1)):
            for use_bias in (True, False):
                y = h.keep(session.linear_adapted(dx, dw, pool, h.ints(choice), db if use_bias else None))
                want = adapted(x, w, bias if use_bias else None, a, b, ranks, scales, choice)
                got = session.download(y)
                np.testing.assert_array_less(np.abs(got - want), 1e-5 * (1 + np.abs(want)))


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("M,N,K,rank", [(1, 1, 8, 1), (1, 577, 1032, 33), (2, 40, 264, 16), (2, 20000, 64, 9), (1, 100, 80, 256), (1, 24, 4096, 16),
                                        (2, 300, 1096, 7), (3, 1536, 576, 8), (2, 1000, 1016, 32)])
def test_linear_of_a_pool_for_one_or_two_rows(session, dtype, M, N, K, rank):
    """Both sides of the rule that gives them one launch; F16 weights; a rank below the pool's; no adapter; no bias."""
    rng = np.random.default_rng(N + K)
    x = rng.standard_normal((M, K)).astype(np.float32)
    bits = oracle.round_f16((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
    w = oracle.widen(bits, oracle.F16)
    a, b, ranks, scales = pool_case(rng, M, N, K, 3, rank, dtype)
    ranks[1], ranks[2] = max(1, rank // 2), 0
    a[1, ranks[1]:], b[1, :, ranks[1]:] = np.nan, np.nan
    a[2], b[2], scales[2] = np.nan, np.nan, np.inf
    bias = rng.standard_normal(N).astype(np.float32)
    with Held(session) as h:
        dw, dx, db = h.keep(session.upload_weight(bits, ffm.STB_F16)), h.f32(x), h.f32(bias)
        pool = device_pool(h, a, b, ranks, scales, dtype)
        for rows in ([0, 1, -7], [1, 1, 0], [-1, 0, 1], [2, 1, 2]):
            rows = np.array(rows[:M])
            for use in (db, None):
                y = h.keep(session.linear_adapted(dx, dw, pool, h.ints(rows), use))
                plain = np.where(rows == 2, -1, rows)  # a slot of rank zero adds nothing
                want = adapted(x, w, bias if use is not None else None, np.nan_to_num(a), np.nan_to_num(b), ranks, scales, plain)
                np.testing.assert_array_less(np.abs(session.download(y) - want), 1e-5 * (1 + np.abs(want)))
        y = h.keep(session.linear_adapted(dx, dw, pool, h.ints(np.full(M, 3))))
        with pytest.raises(ffm.IllegalStateException, match="adapter"):
            session.sync()
        np.testing.assert_array_less(np.abs(session.download(y) - x.astype(np.float64) @ w.T.astype(np.float64)), 2e-5)


@pytest.mark.parametrize("M,N,K", [(96, 2048, 2048), (89, 2048, 2048), (96, 6144, 768), (160, 4096, 1024), (92, 1024, 4096)])
def test_linear_of_a_pool_whose_last_window_takes_more_scratch(session, M, N, K):
    """More than 64 rows whose last window of 64 has 17 to 32: its pieces of the shared product may take more than a whole
    window's."""
    rng = np.random.default_rng(M + N)
    x = rng.standard_normal((M, K)).astype(np.float32)
    bits = oracle.round_bf16((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
    w = oracle.widen(bits, oracle.BF16)
    a, b, ranks, scales = pool_case(rng, M, N, K, 5, 16, "BF16")
    rows = rng.integers(-1, 5, M)
    with Held(session) as h:
        dw, dx = h.keep(session.upload_weight(bits, ffm.STB_BF16)), h.f32(x)
        y = h.keep(session.linear_adapted(dx, dw, device_pool(h, a, b, ranks, scales, "BF16"), h.ints(rows)))
        want = adapted(x, w, None, a, b, ranks, scales, rows)
        np.testing.assert_array_less(np.abs(session.download(y) - want), 1e-5 * (1 + np.abs(want)))


def test_linear_of_a_pool_edges(session):
    """Ranks of zero, negative and behind the pool's; NaN factors behind a slot's rank and in slots that no row names; a
    slot behind the pool; scales of zero and below; empty dimensions."""
    rng = np.random.default_rng(12)
    M, N, K, slots, rank = 6, 256, 128, 5, 16
    x = rng.standard_normal((M, K)).astype(np.float32)
    bits = oracle.round_bf16((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
    w = oracle.widen(bits, oracle.BF16)
    a, b, ranks, scales = pool_case(rng, M, N, K, slots, rank, "F32")
    ranks[:] = [0, -3, 99, 4, 16]
    scales[:] = [1, 1, -0.5, 0.0, 2]
    a[3, 4:], b[3, :, 4:] = np.nan, np.nan
    a[4], b[4] = np.nan, np.nan
    a[0], b[1] = np.nan, np.nan
    rows = np.array([0, 1, 2, 3, -9, 2])
    with Held(session) as h:
        dw, dx = h.keep(session.upload_weight(bits, ffm.STB_BF16)), h.f32(x)
        pool = device_pool(h, a, b, ranks, scales, "F32")
        y = h.keep(session.linear_adapted(dx, dw, pool, h.ints(rows)))
        got, want = session.download(y), adapted(x, w, None, np.nan_to_num(a), np.nan_to_num(b), ranks, scales, rows)
        np.testing.assert_array_less(np.abs(got - want), 1e-5 * (1 + np.abs(want)))
        y = h.keep(session.linear_adapted(dx, dw, pool, h.ints([5, 2, 2, 2, 2 ** 31 - 1, -1])))
        with pytest.raises(ffm.IllegalStateException, match="adapter"):
            session.sync()
        want = adapted(x, w, None, np.nan_to_num(a), np.nan_to_num(b), ranks, scales, [-1, 2, 2, 2, -1, -1])
        np.testing.assert_array_less(np.abs(session.download(y) - want), 1e-5 * (1 + np.abs(want)))
        none = h.keep(session.allocate((0, K)))
        assert session.download(h.keep(session.linear_adapted(none, dw, pool, h.ints(np.zeros(0, int))))).shape == (0, N)


# ------------------------------------------------------------------ the operators together


def step_reference(x, wqkv, bias, pool, rows, qw, kw, pos, caches, tables, heads, kv, width):
    n = len(x)
    fused = adapted(x, wqkv, bias, *pool, rows)
    q = norm_rope(fused[:, :heads * width].reshape(n, heads, width), qw, pos, 1e-6, 10000.0)
    k = norm_rope(fused[:, heads * width:(heads + kv) * width].reshape(n, kv, width), kw, pos, 1e-6, 10000.0)
    v = fused[:, (heads + kv) * width:].reshape(n, kv, width)
    y = []
    for b in range(n):
        caches[b][0].append(k[b])
        caches[b][1].append(v[b])
        y.append(attend(q[b], np.stack(caches[b][0], 1), np.stack(caches[b][1], 1))[0])
    return np.stack(y)


@pytest.mark.parametrize("captured", [False, True])
def test_a_serving_step_of_several_requests(session, captured):
    """Adapted projection -> norm and rotation -> cache write -> attention, four tokens of each of three requests at
    positions of their own (fed as one token per step), in a Float32 paged cache against float64 without pages.  Captured:
    one graph of the step is replayed with new inputs, positions and lengths."""
    import torch
    rng = np.random.default_rng(21)
    n, H, heads, kv, width, page, steps = 3, 192, 6, 2, 64, 4, 9
    N = (heads + 2 * kv) * width
    bits = oracle.round_bf16((rng.standard_normal((N, H)) / np.sqrt(H)).astype(np.float32))
    w = oracle.widen(bits, oracle.BF16)
    bias = rng.standard_normal(N).astype(np.float32)
    pool = pool_case(rng, n, N, H, 3, 8, "BF16")
    rows = np.array([2, -1, 0])
    qw, kw = ((1 + 0.2 * rng.standard_normal(width)).astype(np.float32) for _ in range(2))
    tables, pages = tables_for(rng, [steps] * n, page)
    o = PagedCacheOracle(rng, pages, kv, page, width, "F32")
    xs = rng.standard_normal((steps, n, H)).astype(np.float32)
    with Held(session) as h:
        dw, db = h.keep(session.upload_weight(bits, ffm.STB_BF16)), h.f32(bias)
        dpool, cache = device_pool(h, *pool, "BF16"), h.cache(o)
        dx, dpos, dlen = h.f32(xs[0]), h.ints(np.zeros(n, int)), h.ints(np.ones(n, int))
        drows, dseq, dt, dqw, dkw = h.ints(rows), h.ints(np.arange(n)), h.ints(tables), h.f32(qw), h.f32(kw)
        fused, y = h.keep(session.allocate((n, N))), h.keep(session.allocate((n, heads, width)))
        q, k, v = (h.keep(session.columns(fused, a * width, (c, width))) for a, c in ((0, heads), (heads, kv), (heads + kv, kv)))

        def step():
            session.linear_adapted(dx, dw, dpool, drows, db, out=fused)
            session.qk_norm_rope(q, k, dqw, dkw, dpos, 1e-6, 10000.0, out=(q, k))
            cache.append(k, v, dt, dseq, dpos)
            cache.attend(q, dt, dlen, out=y)

        replay = step
        if captured:
            step()
            session.sync()
            graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(session.stream)
            with torch.cuda.stream(stream):
                graph.capture_begin(capture_error_mode="thread_local")
                step()
                graph.capture_end()

            def replay():
                with torch.cuda.stream(stream):
                    graph.replay()

        caches = [([], []) for _ in range(n)]
        for t in range(steps):
            for dst, src in ((dx, xs[t]), (dpos, np.full(n, t, np.int32)), (dlen, np.full(n, t + 1, np.int32))):
                ffm.call("stb_upload", session.handle, np.ascontiguousarray(src).ctypes.data, src.nbytes, dst.address)
            replay()
            got = session.download(y)
            want = step_reference(xs[t], w, bias, pool, rows, qw, kw, np.full(n, t), caches, tables, heads, kv, width)
            np.testing.assert_array_less(np.abs(got - want), 2e-5 * (1 + np.abs(want)))
        if captured:
            del graph


@pytest.mark.parametrize("rows,N,K,rank", [(6, 1024, 320, 8), (24, 4096, 512, 33), (2, 768, 256, 4)])
def test_steps_behind_one_another_see_what_was_written_before(session, rows, N, K, rank):
    """Calls that start while the one before still runs: 25 steps in a row, the inputs, weights, adapters and tables of each
    written by kernels right before it, give the same bits with a synchronisation after every call and with none."""
    import torch
    heads, kv, width, page, steps = 4, 2, 64, 4, 25
    assert N >= (heads + 2 * kv) * width
    gen = torch.Generator(device="cuda").manual_seed(5)
    f32 = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
    ints = lambda high, *shape: torch.randint(0, high, shape, device="cuda", generator=gen, dtype=torch.int32)
    blocks = -(-(steps + 30) // page)
    start = ints(30, rows)
    new = [dict(x=f32(rows, K), w=(f32(N, K) / K ** 0.5).bfloat16(), a=(f32(3, rank, K) / K ** 0.5).bfloat16(), b=f32(3, N, rank).bfloat16(),
                ranks=ints(rank + 1, 3), slots=ints(4, rows) - 1, bias=f32(N), qw=f32(width), pos=start + t, len=start + t + 1) for t in range(steps)]
    codes = dict(w=ffm.STB_BF16, a=ffm.STB_BF16, b=ffm.STB_BF16, ranks=ffm.STB_I32, slots=ffm.STB_I32, pos=ffm.STB_I32, len=ffm.STB_I32)
    tables = torch.randperm(rows * blocks, device="cuda", generator=gen).int().reshape(rows, blocks)
    seq = torch.arange(rows, device="cuda").int()
    scales, stream = torch.ones(3, device="cuda"), torch.cuda.ExternalStream(session.stream)
    wrap = lambda t, code=ffm.STB_F32: session.wrap(t.data_ptr(), t.shape, code)

    def run(sync):
        now = {k: torch.zeros_like(v) for k, v in new[0].items()}
        pages = [torch.zeros(rows * blocks, kv, page, width, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        fused, y = torch.zeros(rows, N, device="cuda"), torch.zeros(rows, heads, width, device="cuda")
        kept = torch.zeros(steps, *y.shape, device="cuda")
        torch.cuda.synchronize()
        d = {k: wrap(v, codes.get(k, ffm.STB_F32)) for k, v in now.items()}
        cache = session.paged_cache(*[wrap(t, ffm.STB_BF16) for t in pages])
        pool, weight = session.adapter_pool(d["a"], d["b"], d["ranks"], wrap(scales)), session.as_weight(d["w"])
        df, dy, dt, ds = wrap(fused), wrap(y), wrap(tables, ffm.STB_I32), wrap(seq, ffm.STB_I32)
        q, k, v = (session.columns(df, at * width, (n, width)) for at, n in ((0, heads), (heads, kv), (heads + kv, kv)))
        for t in range(steps):
            with torch.cuda.stream(stream):
                for name, value in new[t].items():
                    now[name].copy_(value)
            for call in (lambda: session.linear_adapted(d["x"], weight, pool, d["slots"], d["bias"], out=df),
                         lambda: session.qk_norm_rope(q, k, d["qw"], d["qw"], d["pos"], out=(q, k)),
                         lambda: cache.append(k, v, dt, ds, d["pos"]), lambda: cache.attend(q, dt, d["len"], out=dy)):
                if sync:
                    session.sync()
                call()
            with torch.cuda.stream(stream):
                kept[t].copy_(y)
        session.sync()
        return kept.cpu(), [t.cpu() for t in pages]

    slow, fast = run(True), run(False)
    assert torch.isfinite(slow[0]).all() and (slow[0] != 0).any()
    assert torch.equal(slow[0].view(torch.int32), fast[0].view(torch.int32))
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(slow[1], fast[1]))


def test_captures_allocate_nothing(session):
    """A session's first call inside a capture, and one that would need more scratch, are refused; a graph captured before
    the scratch grew replays on the buffer that it holds.  (The scratch starts at 64 MiB; 64 rows of 131072 outputs take
    two Float32 pieces each, and the terms of x beside them.)"""
    import torch
    rng = np.random.default_rng(23)
    own = ffm.B200Session(0, 4 << 30)
    try:
        with Held(own) as h:
            stream = torch.cuda.ExternalStream(own.stream)

            def projection(M, N, K):
                bits = oracle.round_bf16((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
                x, rows, pool = rng.standard_normal((M, K)).astype(np.float32), rng.integers(-1, 2, M), pool_case(rng, M, N, K, 2, 16, "BF16")
                dw, dpool = h.keep(own.upload_weight(bits, ffm.STB_BF16)), device_pool(h, *pool, "BF16")
                dx, drows, y = h.f32(x), h.ints(rows), h.keep(own.allocate((M, N)))
                return lambda: own.linear_adapted(dx, dw, dpool, drows, out=y), y, adapted(x, oracle.widen(bits, oracle.BF16), None, *pool, rows)

            small, y, want = projection(2, 4096, 4096)
            large, large_y, large_want = projection(64, 131072, 128)
            lengths = [20, 3]
            tables, pages = tables_for(rng, lengths, 16)
            o = PagedCacheOracle(rng, pages, 1, 16, 64, "BF16")
            cache, q = h.cache(o), rng.standard_normal((2, 4, 64)).astype(np.float32)
            dq, dt, dl, dz = h.f32(q), h.ints(tables), h.ints(lengths), h.keep(own.allocate((2, 4, 64)))
            kv = h.f32(rng.standard_normal((2, 1, 64)))

            def captured(calls):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.stream(stream):
                    graph.capture_begin(capture_error_mode="thread_local")
                    own.qk_norm_rope(dq, kv, None, None, dl, out=(dz, kv))
                    calls()
                    graph.capture_end()
                return graph

            def refused(call):
                with pytest.raises(ffm.IllegalStateException):
                    call()

            def first_calls():
                refused(lambda: cache.attend(dq, dt, dl, out=dz))
                refused(lambda: cache.append(kv, kv, dt, dl, dl))
                refused(small)

            del_me = captured(first_calls)
            del del_me
            small()
            own.sync()

            def more_scratch():
                small()
                refused(large)

            graph = captured(more_scratch)
            large()  # grows the scratch
            other = h.f32(rng.standard_normal((1 << 20,)))  # what was freed may be taken again
            kept = own.download(other)
            ffm.call("stb_fill_value", own.handle, y.address, ffm.STB_F32, y.numel, 0.0)
            with torch.cuda.stream(stream):
                graph.replay()
            for got, expected in ((own.download(y), want), (own.download(large_y), large_want)):
                np.testing.assert_array_less(np.abs(got - expected), 1e-5 * (1 + np.abs(expected)))
            assert np.array_equal(own.download(other), kept)
            del graph
    finally:
        own.close()


def test_chunked_prompt_through_a_quantised_cache(session):
    """A prompt's first chunk goes into an E4M3 cache; a later chunk reads it back head-major and attends with
    stb_op_causal_attention; a single new token then attends over the pages: both agree with float64 on what the cache
    stands for."""
    rng = np.random.default_rng(22)
    heads, kv, width, page, first, second = 4, 2, 64, 16, 20, 7
    total = first + second
    tables, pages = tables_for(rng, [total], page)
    o = PagedCacheOracle(rng, pages, kv, page, width, "E4M3")
    k, v = (rng.standard_normal((total, kv, width)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((total, heads, width)).astype(np.float32)
    seq = np.zeros(total, int)
    with Held(session) as h:
        cache, dt = h.cache(o), h.ints(tables)
        for at, n in ((0, first), (first, second)):
            cache.append(h.f32(k[at:at + n]), h.f32(v[at:at + n]), dt, h.ints(seq[:n]), h.ints(at + np.arange(n)))
            for side, x in ((0, k), (1, v)):
                o.append(side, x[at:at + n], tables, seq[:n], at + np.arange(n))
        ks, vs = cache.read(dt, h.ints(seq), h.ints(np.arange(total)), heads_first=True)
        h.keep(ks), h.keep(vs)
        K, V = (h.keep(session.reshape(t, (1, kv, total, width))) for t in (ks, vs))
        Q = h.f32(np.ascontiguousarray(q[first:].transpose(1, 0, 2))[None])
        y = session.download(h.keep(session.causal_attention(Q, K, V, first)))[0]
        lengths = np.array([total])
        one = session.download(h.keep(cache.attend(h.f32(q[-1:]), dt, h.ints(lengths))))[0]
        for t in range(second):
            n = first + t + 1
            want, _, _ = attend(q[first + t], o.rows(0, tables, 0, n), o.rows(1, tables, 0, n))
            np.testing.assert_allclose(y[:, t], want, rtol=0, atol=2e-6)
        np.testing.assert_allclose(one, want, rtol=0, atol=2e-6)


def test_refusals_of_the_library(session):
    """What the C entry points themselves reject, before any launch."""
    with Held(session) as h:
        x = h.keep(session.allocate((4, 256)))
        i = h.keep(session.allocate((8,), ffm.STB_I32))
        a, ia, s = x.address, i.address, session.handle
        before = session.launches

        def cache(**kw):
            f = dict(keys=a, values=a, key_scales=0, value_scales=0, dtype=0, pages=1, page_size=1, kv_heads=1, width=64)
            f.update(kw)
            import ctypes
            return ctypes.byref(ffm.StbPagedCache(*f.values()))

        bad_caches = [dict(keys=0), dict(values=a + 2), dict(dtype=7), dict(dtype=3), dict(key_scales=a), dict(pages=0), dict(page_size=-1),
                      dict(kv_heads=0), dict(width=0), dict(width=513)]
        for kw in bad_caches:
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_op_paged_append", s, cache(**kw), a, 64, 64, a, 64, 64, ia, 1, 1, ia, ia, 1)
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_op_paged_attention", s, cache(**kw), a, 64, 1, ia, 1, 1, ia, a, 64)
        for args in ((0, 64, 64, a, 64, 64, ia, 1, 1, ia, ia, 1), (a + 1, 64, 64, a, 64, 64, ia, 1, 1, ia, ia, 1),
                     (a, 63, 64, a, 64, 64, ia, 1, 1, ia, ia, 2), (a, 64, 64, a, 64, 64, 0, 1, 1, ia, ia, 1),
                     (a, 64, 64, a, 64, 64, ia, -1, 1, ia, ia, 1), (a, 64, 64, a, 64, 64, ia, 1, 1, 0, ia, 1),
                     (a, 64, 64, a, 64, 64, ia, 1, 1, ia, ia + 1, 1), (a, 64, 64, a, 64, 64, ia, 1, 1, ia, ia, -1)):
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_op_paged_append", s, cache(), *args)
        for args in ((0, 64, 1, ia, 1, 1, ia, a, 64), (a, 64, 0, ia, 1, 1, ia, a, 64), (a, 64, 1, ia, 1, 1, 0, a, 64),
                     (a, 64, 1, ia, 1, 1, ia, 0, 64), (a, 60, 1, ia, 2, 1, ia, a, 64), (a, 64, 1, 0, 1, 1, ia, a, 64),
                     (a, 64, 1, ia, 1, -1, ia, a, 64)):
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_op_paged_attention", s, cache(), *args)
        with pytest.raises(ffm.IllegalArgumentException):
            ffm.call("stb_op_paged_attention", s, cache(kv_heads=2), a, 64, 3, ia, 1, 1, ia, a, 64)
        norm = dict(q=a, q_row=64, heads=1, k=a, k_row=64, kv=1, width=64, rows=1, qw=a, kw=a, pos=ia, eps=1e-6, theta=1e4, qo=a, qor=64, ko=a, kor=64)
        for kw in (dict(q=0), dict(q=a + 2), dict(ko=0), dict(width=63), dict(width=514), dict(width=0), dict(rows=-1), dict(heads=-1), dict(pos=0),
                   dict(eps=0.0), dict(eps=float("nan")), dict(theta=0.0), dict(theta=float("inf")), dict(rows=2, q_row=63), dict(qw=a + 1)):
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_op_qk_norm_rope", s, *{**norm, **kw}.values())

        def pool(**kw):
            import ctypes
            f = dict(a=a, b=a, ranks=ia, scales=a, dtype=0, slots=1, max_rank=4)
            f.update(kw)
            return ctypes.byref(ffm.StbAdapterPool(*f.values()))

        for kw in (dict(a=0), dict(b=a + 1), dict(ranks=0), dict(scales=0), dict(dtype=3), dict(slots=0), dict(max_rank=0), dict(max_rank=257)):
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_linear_pool", s, a, a, 0, 0, pool(**kw), ia, a, 1, 8, 8)
        for args in ((0, a, 0, 0, pool(), ia, a, 1, 8, 8), (a, a, 0, 0, pool(), 0, a, 1, 8, 8), (a, a, 0, 0, pool(), ia, a, -1, 8, 8),
                     (a, a, 9, 0, pool(), ia, a, 1, 8, 8), (a, a, 0, 0, None, ia, a, 1, 8, 8), (a, a, 0, 0, pool(), ia, 0, 1, 8, 8)):
            with pytest.raises(ffm.IllegalArgumentException):
                ffm.call("stb_linear_pool", s, *args)
        assert session.launches == before
