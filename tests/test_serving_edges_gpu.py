"""Edges of the serving operators: values that are no numbers, the ends of Float32's range, weights far below the largest.

Tolerances as in test_serving_gpu.py, from the arithmetic there; what differs stands at its test.
"""
import numpy as np
import pytest

import oracle
from scalatorch import ffm
from serving_oracle import PagedCacheOracle, attend, bf16, tables_for
from test_serving_gpu import HALF, Held, adapted, device_pool, pool_case

pytestmark = pytest.mark.gpu
EVERY = ["F32", "BF16", "F16", "E4M3"]
# quiet NaNs as arithmetic on the GPU and on the CPU makes them, of either sign, and one with the lowest payload
NANS = {"F32": (0x7FFFFFFF, 0xFFFFFFFF, 0x7FC00000, 0x7F800001), "BF16": (0x7FFF, 0xFFFF, 0x7FC0, 0x7F81),
        "F16": (0x7FFF, 0xFFFF, 0x7E00, 0x7C01), "E4M3": (0x7F, 0xFF)}


def bits_of(raw):
    return raw.view({4: np.uint32, 2: np.uint16, 1: np.uint8}[raw.itemsize])


def attended(h, o, q, tables, lengths):
    return h.s.download(h.keep(h.cache(o).attend(h.f32(q), h.ints(tables), h.ints(lengths))))


def check_rows(got, o, q, tables, lengths):
    """Every element to the bound of test_serving_gpu.py."""
    for b, n in enumerate(lengths):
        want, mass, score = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
        tol = (np.expm1(2 * (q.shape[2] + 8) * HALF * score) + (n + 16) * 2 * HALF) * mass + 1e-37
        np.testing.assert_array_less(np.abs(got[b].astype(np.float64) - want), tol, err_msg=f"request {b}")


# ------------------------------------------------------------------ NaNs stay NaNs


@pytest.mark.parametrize("width", [64, 33, 256])  # 33: rows of no whole 16 bytes
@pytest.mark.parametrize("dtype", EVERY)
def test_a_nan_of_query_key_or_value_reaches_its_results(session, dtype, width):
    rng = np.random.default_rng(width)
    page, heads, lengths = 16, 4, [40, 40, 40, 40, 1]
    tables, pages = tables_for(rng, lengths, page)
    clean = PagedCacheOracle(rng, pages, 2, page, width, dtype)
    q = rng.standard_normal((5, heads, width)).astype(np.float32)
    for nan in NANS[dtype]:
        o = PagedCacheOracle(np.random.default_rng(1), pages, 2, page, width, dtype)
        for side in range(2):
            o.raw[side], o.scales[side] = clean.raw[side].copy(), clean.scales[side]
        bits_of(o.raw[0])[tables[0, 1], 1, 3, 5] = nan             # a key of kv head 1, request 0
        bits_of(o.raw[1])[tables[1, 0], 0, 2, width - 1] = nan     # a value of kv head 0, request 1
        bits_of(o.raw[1])[tables[4, 0], 1, 0, 0] = nan             # the only token of request 4
        with Held(session) as h:
            got = attended(h, o, q, tables, lengths)
            expected = np.zeros(got.shape, bool)
            expected[0, 2:] = True
            expected[1, :2, width - 1] = True
            expected[4, 2:, 0] = True
            assert np.array_equal(np.isnan(got), expected), (dtype, hex(nan))
            check_rows(got[2:4], o, q[2:4], tables[2:4], lengths[2:4])
    for nan in NANS["F32"]:
        asked = q.copy()
        asked.view(np.uint32)[2, 1, 7] = nan
        with Held(session) as h:
            got = attended(h, clean, asked, tables, lengths)
            expected = np.zeros(got.shape, bool)
            expected[2, 1] = True
            assert np.array_equal(np.isnan(got), expected), (dtype, hex(nan))


@pytest.mark.parametrize("length", [600, 5000])
def test_nans_reach_the_result_across_the_parts_of_a_long_cache(session, length):
    rng = np.random.default_rng(length)
    tables, pages = tables_for(rng, [length], 16)
    o = PagedCacheOracle(rng, pages, 1, 16, 64, "F32")
    q = rng.standard_normal((1, 8, 64)).astype(np.float32)
    for at in (0, length // 2, length - 1):
        before = [r.copy() for r in o.raw]
        bits_of(o.raw[1])[tables[0, at // 16], 0, at % 16, 9] = 0x7FFFFFFF
        with Held(session) as h:
            got = attended(h, o, q, tables, [length])
        assert np.isnan(got[0, :, 9]).all() and np.isfinite(np.delete(got, 9, 2)).all()
        bits_of(o.raw[0])[tables[0, at // 16], 0, at % 16, 0] = 0x7FFFFFFF
        with Held(session) as h:
            assert np.isnan(attended(h, o, q, tables, [length])).all()
        o.raw = before


def test_a_norm_of_nans_reaches_the_attention(session):
    """A head that the norm makes NaN, as it comes out of that kernel, through an F32 cache and as a query."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 2, 64)).astype(np.float32)
    x[1, 1, 5] = np.inf
    o = PagedCacheOracle(rng, 2, 2, 16, 64, "F32")
    with Held(session) as h:
        cache, at, seq, tables = h.cache(o), h.ints([0, 0]), h.ints([0, 1]), h.ints([[0], [1]])
        q, k = (h.keep(t) for t in session.qk_norm_rope(h.f32(x), h.f32(x[::-1].copy()), h.f32(np.ones(64)), h.f32(np.ones(64)), at))
        cache.append(k, h.f32(np.ones((2, 2, 64))), tables, seq, at)
        got = session.download(h.keep(cache.attend(q, tables, h.ints([1, 1]))))
    assert np.isnan(got[0, 1]).all() and np.isnan(got[1, 1]).all() and np.all(got[:, 0] == 1.0)


POOL_FORMS = [(1, 64, 64), (2, 512, 256), (3, 64, 64), (9, 200, 136), (5, 70, 37), (40, 1024, 1024), (70, 1024, 1024)]


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("M,N,K", POOL_FORMS)
def test_a_nan_of_a_factor_or_row_reaches_its_results(session, dtype, M, N, K):
    """In every form of the pool: one launch, three beside the vector product, three beside the tensor cores, 64-row windows."""
    rng = np.random.default_rng(M * N)
    rank = 8
    x = rng.standard_normal((M, K)).astype(np.float32)
    bits = oracle.round_bf16((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
    w = oracle.widen(bits, oracle.BF16)
    a, b, ranks, scales = pool_case(rng, M, N, K, 3, rank, dtype)
    ranks[:] = [rank, rank, rank - 3]
    rows = np.arange(M) % 4 - 1
    rows[0] = 1
    size = {"F32": np.uint32, "BF16": np.uint16, "F16": np.uint16}[dtype]
    with Held(session) as h:
        dw = h.keep(session.upload_weight(bits, ffm.STB_BF16))
        for nan in NANS[dtype]:
            for where in ("a", "b"):
                pool = device_pool(h, a, b, ranks, scales, dtype)
                t = pool.tensors["ab".index(where)]
                raw = session.download_raw(t).view(size).reshape(t.shape).copy()
                raw[(1, 2, K - 1) if where == "a" else (1, N - 1, 2)] = nan
                raw[2, rank - 1 if where == "a" else 0, 0 if where == "a" else rank - 1] = nan  # behind its slot's rank
                ffm.call("stb_upload", session.handle, raw.ctypes.data, raw.nbytes, t.address)
                got = session.download(h.keep(session.linear_adapted(h.f32(x), dw, pool, h.ints(rows))))
                want = adapted(x, w, None, a, b, ranks, scales, rows)
                hit = np.zeros(want.shape, bool)
                hit[rows == 1, 0 if where == "a" else N - 1:] = True
                assert np.array_equal(np.isnan(got), hit), (where, hex(nan))
                np.testing.assert_array_less(np.abs(got - want)[~hit], 1e-5 * (1 + np.abs(want[~hit])))
        pool = device_pool(h, a, b, ranks, scales, dtype)
        for nan in NANS["F32"]:
            bad = x.copy()
            bad.view(np.uint32)[0, K // 2] = nan
            got = session.download(h.keep(session.linear_adapted(h.f32(bad), dw, pool, h.ints(rows))))
            assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


# ------------------------------------------------------------------ the ends of Float32's range

TOP = [3.4028235e38, -3.4028235e38, np.uint32(0x7F7FF000).view(np.float32), np.uint32(0xFF7FF7FF).view(np.float32), 1.7e38, -3.39e38]


@pytest.mark.parametrize("width", [64, 36, 33])
def test_attention_over_float32_values_and_keys_at_the_top_of_the_range(session, width):
    """Values up to Float32's largest beside a weight of one; and keys up to it, whose score takes the whole softmax or none of
    it (3e-5: (width + 8) half steps, twice, of the others' sums of about 3)."""
    rng = np.random.default_rng(width)
    lengths = [1] * len(TOP) + [3] * len(TOP)
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, 1, 16, width, "F32")
    q = rng.standard_normal((len(lengths), 4, width)).astype(np.float32)
    for i, v in enumerate(TOP):
        o.raw[1][tables[i, 0], 0, 0, ::5] = v
        j = len(TOP) + i
        o.raw[0][tables[j, 0], 0, 1, 7] = v
        q[j, :, 7] = 1e-30 * np.arange(1, 5)
    with Held(session) as h:
        got = attended(h, o, q, tables, lengths)
    check_rows(got[:len(TOP)], o, q, tables, lengths[:len(TOP)])
    for j in range(len(TOP), len(lengths)):
        want, mass, _ = attend(q[j], o.rows(0, tables, j, 3), o.rows(1, tables, j, 3))
        np.testing.assert_array_less(np.abs(got[j] - want), 3e-5 * mass + 1e-37)


@pytest.mark.parametrize("M,N,K", POOL_FORMS)
def test_float32_factors_at_the_top_of_the_range(session, M, N, K):
    """One column of A near Float32's largest, beside an x that keeps the products finite."""
    rng = np.random.default_rng(M)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, 0] = 1e-31 * rng.uniform(1, 2, M).astype(np.float32)
    bits = oracle.round_bf16((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
    w = oracle.widen(bits, oracle.BF16)
    a, b, ranks, scales = pool_case(rng, M, N, K, 2, 8, "F32")
    rows = np.arange(M) % 2
    with Held(session) as h:
        dw, dx = h.keep(session.upload_weight(bits, ffm.STB_BF16)), h.f32(x)
        for v in TOP:
            a[:, 0, 0] = v
            got = session.download(h.keep(session.linear_adapted(dx, dw, device_pool(h, a, b, ranks, scales, "F32"), h.ints(rows))))
            want = adapted(x, w, None, a, b, ranks, scales, rows)
            np.testing.assert_array_less(np.abs(got - want), 1e-5 * (1 + np.abs(want)))


# ------------------------------------------------------------------ weights far below the largest


@pytest.mark.parametrize("dtype,width", [("F32", 64), ("BF16", 128), ("F16", 64), ("F16", 128), ("F16", 96), ("F16", 256), ("E4M3", 64), ("E4M3", 128),
                                         ("E4M3", 96), ("E4M3", 256), ("F16", 36)])
@pytest.mark.parametrize("gap", [0, 11, 16, 20, 23, 30, 45])
def test_keys_far_below_one_without_a_value_keep_their_bits(session, dtype, width, gap):
    """A first key `gap` nats above all others whose own value is zero (request 0), or as small as their share of the result
    (request 1), a key like it in the middle (request 2, whose others score alike).  Weights in Float32 keep the rest of
    the result.  Beside the 2e-6 of the norm, the scores' own roundings: a weight moves with its score and the largest one's,
    each within 8 half steps of its sum |q k| / sqrt(width), so 16 half steps of the largest."""
    rng = np.random.default_rng(gap * 7 + width)
    page, lengths, heads = 16, [2001, 2001, 700], 8
    tables, pages = tables_for(rng, lengths, page)
    o = PagedCacheOracle(rng, pages, 1, page, width, dtype)
    q = (0.5 * rng.standard_normal((3, heads, width))).astype(np.float32)
    q[:, :, 0] = np.sqrt(width)
    for b, n in enumerate(lengths):
        k, v = (rng.standard_normal((n, 1, width)).astype(np.float32) for _ in range(2))
        k[:, :, 0] = 0.0
        if b == 2:
            k[:] = k[5]
        first = n // 2 if b == 2 else 0
        k[first] = 0.0
        k[first, 0, 0] = gap
        v[first] *= np.exp(-gap) if b == 1 else 0.0
        for side, x in ((0, k), (1, v)):
            o.append(side, x, tables, np.full(n, b), np.arange(n))
    with Held(session) as h:
        got = attended(h, o, q, tables, lengths)
    check_rows(got, o, q, tables, lengths)
    for b, n in enumerate(lengths):
        want, _, score = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
        off = np.linalg.norm(got[b] - want) / np.linalg.norm(want)
        assert off <= 2e-6 + 16 * HALF * score.max(), (b, off)


@pytest.mark.parametrize("width", [64, 128, 96, 256, 36])
@pytest.mark.parametrize("by", [-6, -12, -20, -40, -80])
def test_small_rows_beside_rows_of_zeros_keep_their_bits(session, width, by):
    """E4M3 rows of zeros carry the scale 2^0, above that of rows of 2^by: every fourth value is zero."""
    rng = np.random.default_rng(width - by)
    lengths = [33, 900]
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, 1, 16, width, "E4M3")
    q = rng.standard_normal((2, 8, width)).astype(np.float32)
    for b, n in enumerate(lengths):
        v = (rng.uniform(1, 2, (n, 1, width)) * 2.0 ** by).astype(np.float32)
        v[::4] = 0.0
        o.append(1, v, tables, np.full(n, b), np.arange(n))
    with Held(session) as h:
        got = attended(h, o, q, tables, lengths)
    check_rows(got, o, q, tables, lengths)
    for b, n in enumerate(lengths):
        want, _, score = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
        assert np.linalg.norm(got[b] - want) <= (2e-6 + 16 * HALF * score.max()) * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", ["F16", "E4M3"])
def test_weights_of_every_size_in_one_cache(session, dtype):
    """Scores spread evenly over 80 nats, rising, falling and shuffled: the running maximum moves, and every tile holds weights
    of many sizes; only the lowest keys have a value in some dimensions."""
    rng = np.random.default_rng(5)
    n, width = 1500, 64
    tables, pages = tables_for(rng, [n] * 3, 16)
    o = PagedCacheOracle(rng, pages, 1, 16, width, dtype)
    q = np.zeros((3, 8, width), np.float32)
    q[:, :, 0] = 8.0
    for b in range(3):
        s = np.linspace(-40, 40, n)
        s = s if b == 0 else (s[::-1] if b == 1 else rng.permutation(s))
        k, v = np.zeros((n, 1, width), np.float32), rng.uniform(1, 2, (n, 1, width)).astype(np.float32)
        k[:, 0, 0] = s
        for d in range(0, 32):
            v[s > 40 - 2 * d, 0, d] = 0.0
        for side, x in ((0, k), (1, v)):
            o.append(side, x, tables, np.full(n, b), np.arange(n))
    with Held(session) as h:
        got = attended(h, o, q, tables, [n] * 3)
    for b in range(3):
        want, mass, score = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
        # each dimension by itself: 40 half steps (22-bit terms, the scores' roundings as above) of its own sum
        np.testing.assert_array_less(np.abs(got[b] - want), (40 + 16 * score.max()) * HALF * mass + 1e-37)


@pytest.mark.parametrize("dtype,width", [("F32", 64), ("BF16", 64), ("F16", 64), ("F16", 128), ("E4M3", 64), ("E4M3", 128), ("E4M3", 256), ("E4M3", 36)])
@pytest.mark.parametrize("spread", [3, 6, 15])
def test_scores_of_any_spread(session, dtype, width, spread):
    """Scores with a standard deviation of `spread` nats: tiles whose weights span much more than F16's exponents; some
    values zero, so that only low weights make a dimension.  Bounds as above."""
    rng = np.random.default_rng(spread + width)
    lengths = [33, 700, 3001, 1]
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, 2, 16, width, dtype)
    q = (spread * rng.standard_normal((4, 10, width))).astype(np.float32)
    for b, n in enumerate(lengths):
        v = rng.standard_normal((n, 2, width)).astype(np.float32)
        v[rng.random(n) < 0.5, :, :width // 2] = 0.0
        o.append(1, v, tables, np.full(n, b), np.arange(n))
    with Held(session) as h:
        got = attended(h, o, q, tables, lengths)
    check_rows(got, o, q, tables, lengths)
    for b, n in enumerate(lengths):
        want, _, score = attend(q[b], o.rows(0, tables, b, n), o.rows(1, tables, b, n))
        assert np.linalg.norm(got[b] - want) <= (2e-6 + 16 * HALF * score.max()) * np.linalg.norm(want)


# ------------------------------------------------------------------ scores of minus infinity


@pytest.mark.parametrize("width", [64, 36, 33, 512])  # whole 16-byte pieces and the others: the answer is the same
@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_keys_whose_scores_overflow_weigh_nothing(session, dtype, width):
    """Finite keys whose score leaves Float32 downwards: the first ones, all but one, all (a row of zeros), none."""
    rng = np.random.default_rng(width)
    lengths = [60, 60, 20, 60]
    tables, pages = tables_for(rng, lengths, 16)
    o = PagedCacheOracle(rng, pages, 1, 16, width, dtype)
    q = (np.abs(rng.standard_normal((4, 4, width))) + 8).astype(np.float32)
    low = np.zeros((4, 60), bool)
    low[0, :23], low[1, :], low[1, 31], low[2] = True, True, False, True
    for b, n in enumerate(lengths):
        k = rng.standard_normal((n, 1, width)).astype(np.float32) / 8
        k[low[b, :n]] = -3e38
        o.append(0, k, tables, np.full(n, b), np.arange(n))
    with Held(session) as h:
        got = attended(h, o, q, tables, lengths)
    for b, n in enumerate(lengths):
        seen = ~low[b, :n]
        k, v = (o.rows(side, tables, b, n)[:, seen] for side in range(2))
        want, mass, score = attend(q[b], k, v)
        tol = (np.expm1(2 * (width + 8) * HALF * score) + (n + 16) * 2 * HALF) * mass + 1e-37
        np.testing.assert_array_less(np.abs(got[b].astype(np.float64) - want), tol, err_msg=f"request {b}")
