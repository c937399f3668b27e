"""Refusals of the serving operators' Python binding, before any native call (no GPU), and their oracle's own answers."""
import numpy as np
import pytest

from scalatorch import ffm
from scalatorch.ffm import STB_BF16, STB_E4M3, STB_F32, STB_I32, STB_U8
from serving_oracle import E4M3, attend, norm_rope, quantise


@pytest.fixture
def s():
    """A session object without a device: native calls on its null handle fail with STATE, so a test that gets an
    IllegalArgumentException was refused before one."""
    session = ffm.B200Session.__new__(ffm.B200Session)
    session.handle, session.device, session.max_bytes, session._closed = None, 0, 1 << 30, False
    return session


def t(s, shape, dtype=STB_F32):
    return s.wrap(1 << 20, shape, dtype)


def test_wrapped_memory_and_views(s):
    x = t(s, (4, 96))
    assert x.nbytes == 4 * 96 * 4 and not x.owner
    c = s.columns(x, 32, (2, 16))
    assert c.shape == (4, 2, 16) and c.row_stride == 96 and c.address == x.address + 32 * 4
    w = s.as_weight(t(s, (8, 4), STB_BF16))
    assert w.shape == (4, 8) and w.transposed_weight
    for bad in (lambda: s.wrap(0, (3,)), lambda: s.wrap(2, (3,)), lambda: s.wrap(16, (-1,)), lambda: s.wrap(16, (1,), 99),
                lambda: s.columns(x, 90, (7,)), lambda: s.columns(x, -1, (7,)), lambda: s.columns(t(s, (2, 2, 2)), 0, (1,)),
                lambda: s.as_weight(t(s, (2, 2, 2))), lambda: s.upload_ints(np.array([1.5])), lambda: s.upload_ints(np.array([1 << 31]))):
        with pytest.raises(ffm.IllegalArgumentException):
            bad()


def test_views_of_columns_are_refused_where_rows_must_be_packed(s):
    c = s.columns(t(s, (4, 96)), 0, (64,))
    for bad in (lambda: s.add(c, c), lambda: s.reshape(c, (256,)), lambda: s.download(c), lambda: s.silu(c), lambda: s.rms_norm(c, t(s, (64,)))):
        with pytest.raises(ffm.IllegalArgumentException):
            bad()


def test_norm_rope_refusals(s):
    q, k, w, p = t(s, (3, 4, 64)), t(s, (3, 2, 64)), t(s, (64,)), t(s, (3,), STB_I32)
    for args in ((t(s, (3, 256)), k, w, w, p), (t(s, (2, 4, 64)), k, w, w, p), (t(s, (3, 4, 32)), k, w, w, p), (q, k, t(s, (32,)), w, p),
                 (q, k, w, t(s, (64,), STB_I32), p), (q, k, w, w, t(s, (4,), STB_I32)), (q, k, w, w, t(s, (3,))), (t(s, (3, 4, 64), STB_BF16), k, w, w, p)):
        with pytest.raises(ffm.IllegalArgumentException):
            s.qk_norm_rope(*args, out=(q, k))
    with pytest.raises(ffm.IllegalArgumentException):
        s.qk_norm_rope(q, k, w, w, p, out=(k, k))
    with pytest.raises(ffm.IllegalStateException):  # a good request reaches the (absent) device
        s.qk_norm_rope(q, k, w, w, p, out=(q, k))


def test_paged_cache_refusals(s):
    shape = (5, 2, 16, 64)
    kv, scale = t(s, shape, STB_E4M3), t(s, shape[:3], STB_U8)
    for args in ((kv, kv), (kv, kv, scale), (kv, kv, scale, t(s, (5, 2, 15), STB_U8)), (kv, t(s, shape, STB_BF16), scale, scale),
                 (t(s, shape), t(s, shape), scale, scale), (t(s, (5, 2, 16)), t(s, (5, 2, 16))), (t(s, (5, 2, 16, 513)),) * 2,
                 (t(s, (0, 2, 16, 64)),) * 2, (t(s, shape, STB_I32),) * 2):
        with pytest.raises(ffm.IllegalArgumentException):
            s.paged_cache(*args)
    c = s.paged_cache(kv, kv, scale, scale)
    x, tab, seq = t(s, (3, 2, 64)), t(s, (2, 4), STB_I32), t(s, (3,), STB_I32)
    for args in ((t(s, (3, 1, 64)), x, tab, seq, seq), (x, t(s, (2, 2, 64)), tab, seq, seq), (x, x, t(s, (8,), STB_I32), seq, seq),
                 (x, x, t(s, (2, 4)), seq, seq), (x, x, tab, t(s, (4,), STB_I32), seq), (x, x, tab, seq, t(s, (3,))), (x, x, tab, t(s, (3, 1), STB_I32), seq)):
        with pytest.raises(ffm.IllegalArgumentException):
            c.append(*args)
    q, n = t(s, (2, 4, 64)), t(s, (2,), STB_I32)
    for args, out in (((t(s, (2, 3, 64)), tab, n), q), ((t(s, (3, 4, 64)), tab, n), q), ((t(s, (2, 4, 32)), tab, n), q), ((q, tab, seq), q),
                      ((q, tab, n), t(s, (2, 4, 32)))):
        with pytest.raises(ffm.IllegalArgumentException):
            c.attend(*args, out=out)
    with pytest.raises(ffm.IllegalArgumentException):
        c.read(tab, seq, seq, out=(x, t(s, (2, 3, 64))))
    with pytest.raises(ffm.IllegalStateException):
        c.read(tab, seq, seq, out=(t(s, (2, 3, 64)), t(s, (2, 3, 64))), heads_first=True)
    kv._alive[0] = False
    with pytest.raises(ffm.IllegalStateException, match="released"):
        c.attend(q, tab, n, out=q)


def test_adapter_pool_refusals(s):
    a, b, r, sc = t(s, (3, 8, 32)), t(s, (3, 48, 8)), t(s, (3,), STB_I32), t(s, (3,))
    for args in ((a, t(s, (3, 48, 8), STB_BF16), r, sc), (a, t(s, (2, 48, 8)), r, sc), (a, t(s, (3, 48, 4)), r, sc), (a, b, sc, sc), (a, b, r, r),
                 (t(s, (3, 257, 32)), t(s, (3, 48, 257)), r, sc), (t(s, (8, 32)), b, r, sc)):
        with pytest.raises(ffm.IllegalArgumentException):
            s.adapter_pool(*args)
    pool = s.adapter_pool(a, b, r, sc)
    w, x, rows, y = s.as_weight(t(s, (48, 32), STB_BF16)), t(s, (5, 32)), t(s, (5,), STB_I32), t(s, (5, 48))
    for args, out in (((x, w, pool, t(s, (4,), STB_I32)), y), ((t(s, (5, 33)), w, pool, rows), y), ((x, s.as_weight(t(s, (40, 32), STB_BF16)), pool, rows), y),
                      ((x, w, pool, rows, t(s, (47,))), y), ((x, w, pool, rows), x), ((x, t(s, (48, 32), STB_BF16), pool, rows), y)):
        with pytest.raises(ffm.IllegalArgumentException):
            s.linear_adapted(*args, out=out)
    with pytest.raises(ffm.IllegalStateException):
        s.linear_adapted(x, w, pool, rows, out=y)


def test_operands_that_are_no_tensors(s):
    a, i = np.zeros((3, 2, 64), np.float32), np.zeros(3, np.int32)
    kv = t(s, (5, 2, 16, 64))
    c, pool = s.paged_cache(kv, kv), s.adapter_pool(t(s, (3, 8, 32)), t(s, (3, 48, 8)), t(s, (3,), STB_I32), t(s, (3,)))
    for bad in (lambda: s.qk_norm_rope(a, a, None, None, i, out=(a, a)), lambda: c.append(a, a, i[None], i, i), lambda: c.read(i[None], i, i, out=(a, a)),
                lambda: c.attend(a, i[None], i, out=a), lambda: s.linear_adapted(a, a, pool, i), lambda: s.linear_adapted(a, a, None, i)):
        with pytest.raises(ffm.IllegalArgumentException):
            bad()


def test_the_oracles_known_answers():
    assert E4M3[0x7E] == 448.0 and E4M3[1] == 2.0 ** -9 and E4M3[0x38] == 1.0 and np.isnan(E4M3[0x7F])
    q, e = quantise(np.array([[448.0, 1.0, 0.0, -17.0], [449.0, 1.0, 0.0, -17.0], [0.0, 0.0, 0.0, 0.0], [np.inf, 2.0, np.nan, -2.0]]))
    assert list(e) == [127, 128, 127, 127 - 7]
    assert list(q[0]) == [0x7E, 0x38, 0, 0x80 | 0x58] and q[1][0] == 0x76 and list(q[2]) == [0] * 4
    assert q[3][0] & 127 == 127 and E4M3[q[3][1]] == 256.0 and q[3][2] & 127 == 127
    x = np.array([[[3.0, 4.0]]])
    np.testing.assert_allclose(norm_rope(x, None, [0], 1e-6, 1e4), x)
    np.testing.assert_allclose(norm_rope(x, [1, 1], [0], 1e-300, 1e4), x / np.sqrt(12.5))
    np.testing.assert_allclose(norm_rope(x, None, [1], 1e-6, 1e4)[0, 0], [3 * np.cos(1) - 4 * np.sin(1), 4 * np.cos(1) + 3 * np.sin(1)])
    y, _, _ = attend(np.array([[2.0, 0.0]]), np.array([[[0.0, 1.0], [0.0, 5.0]]]), np.array([[[1.0, 2.0], [3.0, 4.0]]]))
    np.testing.assert_allclose(y, [[2.0, 3.0]])
    assert np.all(attend(np.ones((1, 2)), np.zeros((1, 0, 2)), np.zeros((1, 0, 2)))[0] == 0)


def test_a_column_is_no_packed_vector(s):
    """One column of a matrix has a weight's or a bias's shape, but its elements lie apart."""
    q, k, p = t(s, (3, 4, 64)), t(s, (3, 2, 64)), t(s, (3,), STB_I32)
    w, apart = t(s, (64,)), s.columns(t(s, (64, 5)), 2, ())
    assert apart.shape == (64,) and apart.row_stride == 5
    for weights in ((apart, w), (w, apart)):
        with pytest.raises(ffm.IllegalArgumentException, match="packed"):
            s.qk_norm_rope(q, k, *weights, p, out=(q, k))
    pool = s.adapter_pool(t(s, (3, 8, 32)), t(s, (3, 48, 8)), t(s, (3,), STB_I32), t(s, (3,)))
    x, rows, y = t(s, (5, 32)), t(s, (5,), STB_I32), t(s, (5, 48))
    bias = s.columns(t(s, (48, 9)), 0, ())
    with pytest.raises(ffm.IllegalArgumentException, match="packed"):
        s.linear_adapted(x, s.as_weight(t(s, (48, 32), STB_BF16)), pool, rows, bias, out=y)
