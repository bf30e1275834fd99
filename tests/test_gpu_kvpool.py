"""A cache in pages: rows quantised into it and read back, bit for bit, and attention over it against 64-bit arithmetic."""
import ctypes as C

import numpy as np
import pytest

from tests import kvpool_plain as plain
from tests.kvpool_plain import BF16, F16, F32, Cache, Device, from_type, held, rounded, to_type

pytestmark = pytest.mark.gpu
DTYPE = {F32: np.float32, F16: np.float16, BF16: np.uint16}
KV = ("i8", "e4m3", "f16", "bf16")


@pytest.fixture()
def dev():
    from llama2_rs import _lib
    assert _lib.lib().l2_device_count() >= 1, "no HIP device: the GPU tests cannot run"
    d = Device()
    yield d
    d.close()


def _values(rng, shape):
    """Rows of different magnitudes, with values on the borders between codes, zeros, and rows of nothing else."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,)) * 3)
    x = x.astype(np.float32)
    flat = x.reshape(-1, shape[-1])
    for r in range(0, len(flat), 7):  # whole and half steps of the row's largest value
        flat[r] = np.round(flat[r] / np.abs(flat[r]).max() * 254) / 254 * np.float32(2.0 ** rng.integers(-8, 8))
    flat[::11, 3] = 0.0
    if len(flat) > 13:
        flat[13] = 0.0
        flat[12] = 1e-30
        flat[9, 5] = -flat[9, 4]
    return flat.reshape(shape)


def _read(c, dev, rows, t, batch=None, n=None, fill=7.0):
    n = sum(rows) if n is None else n
    b = batch if batch is not None else c.batch(rows)
    out = [dev.put(to_type(np.full((n, c.kv_heads, c.head_size), fill, np.float32), t)) for _ in "kv"]
    c.pool.read(c.layer, b, out[0], out[1], t)
    return [from_type(dev.get(p, (n, c.kv_heads, c.head_size), DTYPE[t]), t) for p in out]


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("page,kv_heads,head_size", [(16, 3, 128), (64, 8, 64), (256, 1, 128), (32, 5, 64)])
def test_written_rows_read_back(dev, kv, t, page, kv_heads, head_size):
    lengths = [1, 37, 0, 300, 16, 64, 130]
    c = Cache(dev, kv, page, kv_heads, head_size, lengths, seed=page)
    rng = np.random.default_rng(page + kv_heads)
    shape = (sum(lengths), kv_heads, head_size)
    k, v = _values(rng, shape), _values(rng, shape)
    if t == F16:
        k, v = np.clip(k, -60000, 60000), np.clip(v, -60000, 60000)
    c.fill(k, v, t)
    for out in (F32, t):
        got = _read(c, dev, lengths, out)
        for g, want in zip(got, (c.k, c.v)):
            np.testing.assert_array_equal(g, rounded(want, out))
    c.close()


@pytest.mark.parametrize("kv", KV)
def test_rows_that_follow_one_another(dev, kv):
    """A prompt, then chunks and single tokens of some sequences, others without a row: what is there before stays."""
    rng = np.random.default_rng(5)
    most = [75, 40, 20, 33]
    c = Cache(dev, kv, 16, 2, 128, most, seed=2)
    want = [np.zeros((m, 2, 128), np.float32) for m in most]
    now = [0, 0, 0, 0]
    for rows in ([50, 3, 0, 17], [1, 1, 1, 0], [0, 30, 18, 15], [23, 0, 1, 1], [1, 6, 0, 0]):
        now = [a + b for a, b in zip(now, rows)]
        x = [rng.standard_normal((sum(rows), 2, 128)).astype(np.float32) for _ in "kv"]
        b = c.batch(rows, now, first=2, behind=3)
        pad = [np.concatenate([np.full((2, 2, 128), np.nan, np.float32), y, np.full((3, 2, 128), np.nan, np.float32)]) for y in x]
        c.pool.write(0, b, dev.put(pad[0]), dev.put(pad[1]), F32)
        at = 0
        for i, n in enumerate(rows):
            want[i][now[i] - n:now[i]] = held(x[0][at:at + n], kv)
            at += n
        got = _read(c, dev, now, F32, c.batch(now, now))[0]
        np.testing.assert_array_equal(got, np.concatenate([w[:n] for w, n in zip(want, now)]))
    # only some of the last positions
    rows = [5, 0, 2, 9]
    got = _read(c, dev, rows, F32, c.batch(rows, now, first=1, behind=2), n=19)[0]
    np.testing.assert_array_equal(got[1:17], np.concatenate([w[n - r:n] for w, n, r in zip(want, now, rows)]))
    assert np.all(got[0] == 7.0) and np.all(got[17:] == 7.0)
    c.close()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_strides_and_addresses(dev, kv, t):
    """Rows of a wider array (fused q|k|v), at odd strides and addresses that are multiples of the type's size alone."""
    rng = np.random.default_rng(3)
    lengths, H, D = [21, 34], 3, 64
    c = Cache(dev, kv, 16, H, D, lengths)
    n = sum(lengths)
    for wide, off in ((2 * H * D + 5, 1), (2 * H * D + 8, 8)):
        x = rng.standard_normal((n, wide)).astype(np.float32)
        p, size = dev.put(to_type(np.concatenate([np.zeros(off, np.float32), x.reshape(-1)]), t)), plain.BYTES[t]
        c.pool.write(0, c.batch(lengths), p + off * size, p + (off + H * D) * size, t, wide, wide)
        want = [held(rounded(x[:, a:a + H * D].reshape(n, H, D), t), kv) for a in (0, H * D)]
        out = dev.put(to_type(np.full(off + n * wide, 7.0, np.float32), t))
        c.pool.read(0, c.batch(lengths), out + off * size, out + (off + H * D) * size, t, wide, wide)
        got = from_type(dev.get(out, (off + n * wide,), DTYPE[t]), t)
        assert np.all(got[:off] == 7.0)
        got = got[off:].reshape(n, wide)
        for g, w in zip((got[:, :H * D], got[:, H * D:2 * H * D]), want):
            np.testing.assert_array_equal(g.reshape(n, H, D), rounded(w, t))
        assert np.all(got[:, 2 * H * D:] == 7.0)
    c.close()


@pytest.mark.parametrize("kv", KV)
def test_values_that_are_not_finite_and_pages_that_are_not_there(dev, kv):
    rng = np.random.default_rng(8)
    lengths = [40, 40]
    c = Cache(dev, kv, 16, 2, 64, lengths)
    k, v = (rng.standard_normal((80, 2, 64)).astype(np.float32) for _ in "kv")
    k[3, 0, 5], k[4, 1, 0], v[5, 0, 63], v[70, 1, 2] = np.nan, np.inf, -np.inf, np.nan
    k[6], v[6] = 3e38, -3e38
    c.fill(k, v)
    got = _read(c, dev, lengths, F32)
    np.testing.assert_array_equal(got[0], c.k)
    np.testing.assert_array_equal(got[1], c.v)
    # rows of pages outside the pool, and of positions below zero, are not written and read as zeros; others are
    table = c.table.copy()
    table[0, 1], table[1, 0] = c.n_pages, -5
    rows = [40, 45]
    x = rng.standard_normal((85, 2, 64)).astype(np.float32)
    b = c.batch(rows, lengths, table=table)
    c.pool.write(0, b, dev.put(x), dev.put(-x), F32)
    there = np.ones(85, bool)
    there[16:32] = False
    there[40:45] = False
    there[45:61] = False
    got = _read(c, dev, rows, F32, b, 85)
    want = np.where(there[:, None, None], held(x, kv), 0)
    np.testing.assert_array_equal(got[0], want)
    np.testing.assert_array_equal(got[1], -want)
    old = _read(c, dev, lengths, F32)[0]  # what the pages hold that were not named
    np.testing.assert_array_equal(old[16:32], c.k[16:32])
    np.testing.assert_array_equal(old[40:56], c.k[40:56])
    c.close()


def test_layers_are_apart(dev):
    rng = np.random.default_rng(1)
    c = Cache(dev, "i8", 32, 2, 128, [50], layers=3)
    x = rng.standard_normal((3, 2, 50, 2, 128)).astype(np.float32)
    for layer in range(3):
        c.pool.write(layer, c.batch([50]), dev.put(x[layer, 0]), dev.put(x[layer, 1]), F32)
    for layer in range(3):
        c.layer = layer
        got = _read(c, dev, [50], F32)
        for g, w in zip(got, x[layer]):
            np.testing.assert_array_equal(g, held(w, "i8"))
    c.close()


# ---- attention ------------------------------------------------------------------------------------------------


def _filled(dev, kv, page, kv_heads, head_size, lengths, seed=0, t=F32, **more):
    c = Cache(dev, kv, page, kv_heads, head_size, lengths, seed=seed, **more)
    rng = np.random.default_rng(seed + 1)
    shape = (sum(lengths), kv_heads, head_size)
    k = rng.standard_normal(shape) * np.exp(0.4 * rng.standard_normal(shape[1:]))
    v = rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[:2] + (1,)))
    c.fill(k.astype(np.float32), v.astype(np.float32), t)
    return c, rng


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("page,kv_heads,group,head_size", [(16, 2, 1, 128), (64, 1, 8, 128), (32, 3, 5, 64), (256, 2, 2, 64), (128, 1, 16, 128)])
def test_single_tokens(dev, kv, t, page, kv_heads, group, head_size):
    lengths = [1, 2, 15, 16, 17, 33, 63, 64, 65, 127, 300, 519]
    c, rng = _filled(dev, kv, page, kv_heads, head_size, lengths, seed=page + group, t=t)
    rows, heads = [1] * len(lengths), kv_heads * group
    q = rng.standard_normal((len(lengths), heads, head_size)).astype(np.float32)
    for window, sinks in ((0, 0), (7, 0), (64, 4), (100, 70)):
        got = c.attend(q, rows, t, heads, window, sinks)
        c.check(got, q, rows, t, heads, window, sinks)
    c.close()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("page,kv_heads,group,head_size", [(16, 2, 1, 128), (64, 1, 8, 128), (32, 1, 3, 64)])
def test_chunks(dev, kv, t, page, kv_heads, group, head_size):
    lengths, rows = [5, 40, 130, 200, 64, 1], [5, 33, 130, 7, 64, 1]
    c, rng = _filled(dev, kv, page, kv_heads, head_size, lengths, seed=page + group, t=t)
    heads = kv_heads * group
    q = rng.standard_normal((sum(rows), heads, head_size)).astype(np.float32)
    for window, sinks in ((0, 0), (9, 3), (70, 20)):
        got = c.attend(q, rows, t, heads, window, sinks)
        c.check(got, q, rows, t, heads, window, sinks)
    c.close()


@pytest.mark.parametrize("kv,t", [("i8", F32), ("e4m3", BF16), ("f16", F16), ("bf16", BF16)])
def test_long_contexts(dev, kv, t):
    """Single tokens and a chunk behind thousands of positions, in one call."""
    lengths, rows = [3001, 777, 4500], [1, 20, 2]
    c, rng = _filled(dev, kv, 64, 1, 128, lengths, seed=4, t=t)
    q = 2 * rng.standard_normal((sum(rows), 4, 128)).astype(np.float32)
    for window, sinks in ((0, 0), (1000, 2)):
        got = c.attend(q, rows, t, 4, window, sinks)
        c.check(got, q, rows, t, 4, window, sinks)
    c.close()


@pytest.mark.parametrize("kv,t", [("i8", F16), ("i8", F32), ("e4m3", BF16), ("f16", F16), ("f16", F32), ("bf16", BF16), ("bf16", F32)])
@pytest.mark.parametrize("group,most", [(1, 64), (5, 12), (8, 4), (8, 9), (32, 1), (40, 1), (72, 1)])
def test_a_few_tokens_each(dev, kv, t, group, most):
    """Up to 17, 32, 64 and some more query rows per kv head, which are blocks of 16, of one kernel or the other."""
    rows = [most, 1, (most + 1) // 2, most, 0]
    lengths = [most, 500, 333, 70, 20]
    c, rng = _filled(dev, kv, 16, 2, 64 if group == 5 else 128, lengths, seed=group, t=t)
    q = rng.standard_normal((sum(rows) + 3, 2 * group, c.head_size)).astype(np.float32)
    for window, sinks in ((0, 0), (90, 5)):
        got = c.attend(q, None, t, 2 * group, window, sinks, batch=c.batch(rows, first=1, behind=2))
        c.check(got, q, rows, t, 2 * group, window, sinks, first=1)
    c.close()


@pytest.mark.parametrize("kv,t", [("i8", F16), ("e4m3", F32), ("f16", BF16), ("bf16", F32)])
def test_groups_that_do_not_divide_a_tile(dev, kv, t):
    """Chunks of several tiles of rows whose borders lie inside a token's heads, behind many tiles that all of them see."""
    lengths, rows = [700, 1000], [111, 38]
    c, rng = _filled(dev, kv, 32, 1, 128, lengths, seed=8, t=t)
    q = rng.standard_normal((sum(rows), 7, 128)).astype(np.float32)
    for window, sinks in ((0, 0), (333, 5)):
        got = c.attend(q, rows, t, 7, window, sinks)
        c.check(got, q, rows, t, 7, window, sinks)
    c.close()


@pytest.mark.parametrize("kv", ["i8", "bf16"])
def test_pages_past_32_bits(dev, kv):
    """Keys of more than 2^32 bytes, and sequences in their last pages."""
    lengths, rows, heads = [600, 290], [1, 20], 32
    c = Cache(dev, kv, 256, heads, 128, lengths, extra_pages=4200)
    assert c.pool.nbytes > 2 * 2 ** 32
    c.table[0] = c.n_pages - 1 - np.arange(c.max_pages)
    c.table[1, :2] = [0, c.n_pages - 1 - c.max_pages]
    rng = np.random.default_rng(9)
    k, v = (rng.standard_normal((sum(lengths), heads, 128)).astype(np.float32) for _ in "kv")
    c.fill(k, v)
    for got, want in zip(_read(c, dev, lengths, F32), (c.k, c.v)):
        np.testing.assert_array_equal(got, want.astype(np.float32))
    q = rng.standard_normal((sum(rows), heads, 128)).astype(np.float32)
    c.check(c.attend(q, rows, F32, heads), q, rows, F32, heads)
    c.close()


@pytest.mark.parametrize("kv,t", [("i8", F32), ("e4m3", F16), ("f16", F32), ("bf16", F32), ("bf16", F16), ("f16", BF16)])
def test_rows_that_see_nothing(dev, kv, t):
    """No positions, no rows, more rows than positions, and rows of no sequence."""
    lengths = [20, 0, 6, 0, 33]
    c, rng = _filled(dev, kv, 16, 2, 64, lengths, t=t)
    for rows in ([3, 2, 9, 0, 1], [1, 1, 1, 0, 1], [0, 0, 0, 0, 1], [20, 40, 20, 0, 33]):
        b = c.batch(rows, first=2, behind=3)
        q = rng.standard_normal((sum(rows) + 5, 4, 64)).astype(np.float32)
        got = c.attend(q, rows, t, 4, batch=b)
        c.check(got, q, rows, t, 4, first=2)
    c.close()


@pytest.mark.parametrize("kv", KV)
def test_pages_that_are_not_there_are_not_seen(dev, kv):
    lengths, rows = [100, 90, 200], [1, 30, 200]
    c, rng = _filled(dev, kv, 16, 1, 128, lengths)
    q = rng.standard_normal((sum(rows), 2, 128)).astype(np.float32)
    table = c.table.copy()
    missing = [(0, 0), (0, 3), (0, 6), (1, 2), (1, 5), (2, 0), (2, 7), (2, 12)]
    for i, p in missing:
        table[i, p] = -1 if p % 2 else c.n_pages + p
    got = c.attend(q, rows, F32, 2, batch=c.batch(rows, table=table))
    c.check(got, q, rows, F32, 2, missing=missing)
    # the pages outside of every row's window need not be there
    table = c.table.copy()
    table[0, 1:3], table[1, 1], table[2, 9:] = -1, 1 << 30, c.table[2, 9:]
    for window, sinks in ((40, 5),):
        keep = table.copy()
        keep[2] = c.table[2]
        got = c.attend(q, rows, F32, 2, window, sinks, batch=c.batch(rows, table=keep))
        c.check(got, q, rows, F32, 2, window, sinks, missing=[(1, 1)])
    c.close()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("what", ["nan", "inf", "big"])
def test_what_is_not_seen_has_no_influence(dev, kv, t, what):
    """NaN, infinities and huge values at positions that some rows or none see: rows that do not are as if those were not there."""
    lengths, rows = [70, 150], [70, 20]
    c, rng = _filled(dev, kv, 32, 1, 128, lengths, t=t)
    k, v = (rng.standard_normal((220, 1, 128)).astype(np.float32) for _ in "kv")
    bad = {"nan": np.nan, "inf": np.inf, "big": 60000.0}[what]
    k[50], v[60, 0, 7] = bad, bad          # of the first sequence: rows behind them see them
    v[62], k[69] = -bad, bad
    k[70 + 20], v[70 + 25] = bad, -bad     # of the second, before the windows of its rows
    v[70 + 149] = bad                      # its last row's own
    c.fill(k, v, t)
    q = rng.standard_normal((90, 2, 128)).astype(np.float32)
    q[3, 1, 4] = np.nan
    got = c.attend(q, rows, t, 2, window=48, sinks=3)
    clean = np.isfinite(got).all(-1)
    qq, kk, vv = rounded(q, t), c.k, c.v
    at = 0
    for i, n in enumerate(rows):
        for j in range(n):
            m = plain.seen(lengths[i] - n + j, lengths[i], 48, 3)
            ks, vs = kk[c.rows_of(i)][m][:, 0], vv[c.rows_of(i)][m][:, 0]
            for h in range(2):
                fine = np.isfinite(ks).all() and np.isfinite(vs).all() and np.isfinite(qq[at, h]).all()
                if fine:
                    want, size, most = plain.attention_row(qq[at, h], ks, vs, 128 ** -0.5)
                    bound = plain.attention_bound(kv, t, size, most, int(m.sum()), 128, want)
                    assert np.all(np.abs(got[at, h] - want) <= bound), (i, j, h)
                elif not np.isfinite(ks).all() or not np.isfinite(qq[at, h]).all():
                    assert np.isnan(got[at, h]).all() or not np.isfinite(plain.attention_row(qq[at, h], ks, vs, 1.0)[0]).all(), (i, j, h)
                else:  # a value that is not finite makes its dimension so, and in 8 bits its row
                    assert not np.isfinite(got[at, h][~np.isfinite(vs).all(0)]).any(), (i, j, h)
            at += 1
    assert clean.any() and (what == "big" or not clean.all())
    # what pages hold behind the last position, of sequences that had them before
    c.fill(np.full((220, 1, 128), bad, np.float32), np.full((220, 1, 128), -bad, np.float32), t)
    short, srows = [33, 65], [33, 2]
    k2, v2 = (rng.standard_normal((98, 1, 128)).astype(np.float32) for _ in "kv")
    c.pool.write(0, c.batch(short, short), dev.put(to_type(k2, t)), dev.put(to_type(v2, t)), t)
    c.k[:33], c.k[70:135] = held(rounded(k2, t), kv)[:33], held(rounded(k2, t), kv)[33:]
    c.v[:33], c.v[70:135] = held(rounded(v2, t), kv)[:33], held(rounded(v2, t), kv)[33:]
    q = rng.standard_normal((35, 2, 128)).astype(np.float32)
    got = c.attend(q, srows, t, 2, batch=c.batch(srows, short))
    c.check(got, q, srows, t, 2, lengths=short)
    c.close()


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("t", [F32, F16])
def test_rows_of_very_different_scales(dev, kv, t):
    """Magnitudes of values from 2^-50 to 2^50 in one sequence: rows that see only small ones keep their accuracy."""
    lengths, rows = [200, 130], [200, 1]
    c, rng = _filled(dev, kv, 32, 1, 64, lengths)
    n = sum(lengths)
    k = 0.3 * rng.standard_normal((n, 1, 64)).astype(np.float32)
    v = rng.standard_normal((n, 1, 64)).astype(np.float32)
    v[:200] *= np.exp2(np.linspace(-50, 13 if t == F16 else 50, 200)).astype(np.float32)[:, None, None]
    v[200:] *= np.exp2(rng.integers(-50, -20, (130, 1, 1))).astype(np.float32)
    v[17] = 0
    c.fill(k, v)
    q = rng.standard_normal((sum(rows), 2, 64)).astype(np.float32)
    for window, sinks in ((0, 0), (20, 2)):
        got = c.attend(q, rows, t, 2, window, sinks)
        c.check(got, q, rows, t, 2, window, sinks)
    c.close()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_magnitudes_of_queries(dev, kv, t):
    """Queries from the smallest numbers of their type to large ones, and scores that leave one position everything."""
    lengths, rows = [90], [30]
    c, rng = _filled(dev, kv, 16, 1, 64, lengths, t=t)
    q = rng.standard_normal((30, 1, 64)).astype(np.float32)
    q *= np.exp2(np.linspace(-24 if t == F16 else -120, 6, 30)).astype(np.float32)[:, None, None]
    q[4] = 0
    got = c.attend(q, rows, t, 1)
    c.check(got, q, rows, t, 1)
    c.close()


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_attention_strides_and_in_place(dev, t):
    lengths, rows, H, D = [50, 20], [9, 20], 4, 64
    c, rng = _filled(dev, "i8", 16, 2, D, lengths, t=t)
    n, size = sum(rows), plain.BYTES[t]
    for wide, off in ((2 * H * D + 3, 1), (3 * H * D, 8)):
        x = rng.standard_normal((n, wide)).astype(np.float32)
        p = dev.put(to_type(np.concatenate([np.zeros(off, np.float32), x.reshape(-1)]), t))
        b = c.batch(rows)
        need = c.pool.attention_workspace(b, H, t)
        work = dev.empty(need)
        out = dev.put(to_type(np.full(off + n * wide, 7.0, np.float32), t))
        c.pool.attention(0, b, p + off * size, out + off * size, H, t, workspace=work, workspace_bytes=need, q_stride=wide, out_stride=wide)
        got = from_type(dev.get(out, (off + n * wide,), DTYPE[t]), t)
        q = x[:, :H * D].reshape(n, H, D)
        c.check(got[off:].reshape(n, wide)[:, :H * D].reshape(n, H, D), q, rows, t, H)
        assert np.all(got[:off] == 7.0) and np.all(got[off:].reshape(n, wide)[:, H * D:] == 7.0)
        c.pool.attention(0, b, p + off * size, p + off * size, H, t, workspace=work, workspace_bytes=need, q_stride=wide, out_stride=wide)
        again = from_type(dev.get(p, (off + n * wide,), DTYPE[t]), t)
        np.testing.assert_array_equal(again[off:].reshape(n, wide)[:, :H * D], got[off:].reshape(n, wide)[:, :H * D])
        np.testing.assert_array_equal(again[off:].reshape(n, wide)[:, H * D:], rounded(x, t)[:, H * D:])
    c.close()


def test_scale(dev):
    c, rng = _filled(dev, "f16", 16, 2, 64, [77])
    q = rng.standard_normal((5, 2, 64)).astype(np.float32)
    for scale in (1.0, 0.01, 1e-30, 3.0):
        got = c.attend(q, [5], F32, 2, scale=scale)
        c.check(got, q, [5], F32, 2, scale=float(np.float32(scale)))
    c.close()


def _graph(rt, stream, call):
    graph, gexec = C.c_void_p(), C.c_void_p()
    assert rt.hipStreamBeginCapture(stream, 0) == 0            # hipStreamCaptureModeGlobal
    try:
        call()
    finally:
        assert rt.hipStreamEndCapture(stream, C.byref(graph)) == 0
    n = C.c_size_t()
    assert rt.hipGraphGetNodes(graph, None, C.byref(n)) == 0 and n.value >= 1
    nodes = (C.c_void_p * n.value)()
    assert rt.hipGraphGetNodes(graph, nodes, C.byref(n)) == 0
    for node in nodes:
        kind = C.c_int()
        assert rt.hipGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
        assert kind.value == 0, f"graph node of type {kind.value}: only kernel nodes are expected"
    assert rt.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
    return graph, gexec


@pytest.mark.parametrize("kv,t", [("i8", F32), ("e4m3", BF16), ("bf16", BF16)])
def test_a_step_captured_and_replayed(dev, kv, t):
    """Rows written, attended and sampled in one graph, the pool's first calls among them, replayed with other rows, lengths and
    pages, with eager calls between: every replay equals the eager calls, and the formula."""
    from llama2_rs import ops
    rt, H, KVH, D, V = dev.rt, 4, 2, 64, 500
    top = [200, 90, 33]
    c = Cache(dev, kv, 16, KVH, D, top, layers=1)
    stream = C.c_void_p()
    assert rt.hipStreamCreate(C.byref(stream)) == 0
    rng = np.random.default_rng(6)
    n = 12
    dk, dv, dq, out = (dev.empty(n * h * D * 4) for h in (KVH, KVH, H, H))
    starts, lengths, table = dev.empty(16), dev.empty(16), dev.empty(c.table.nbytes)
    b = ops.KvBatch(starts, lengths, table, 3, c.max_pages, n, 8, 200)
    need = c.pool.attention_workspace(b, H, t, 50, 4)
    work = dev.empty(need)
    logits, ids, u = dev.empty(3 * V * 4), dev.empty(16), dev.put(np.array([0.1, 0.5, 0.9], np.float32))
    top_p = dev.put(np.array([0.9, 1.0, 0.5], np.float32))

    def step(s):
        c.pool.write(0, b, dk, dv, t, stream=s)
        c.pool.attention(0, b, dq, out, H, t, window=50, sinks=4, workspace=work, workspace_bytes=need, stream=s)
        ops.sample_device(logits, 3, V, ids, u, top_p=top_p, stream=s)

    graph, gexec = _graph(rt, stream, lambda: step(stream.value))
    c.k = np.zeros((sum(top), KVH, D), np.float32)
    c.v = np.zeros_like(c.k)
    now = [0, 0, 0]
    first = np.cumsum([0] + top)
    for rows in ([8, 3, 1], [1, 1, 1], [0, 8, 1], [1, 0, 7], [4, 1, 1], [1, 1, 1]):
        now = [a + x for a, x in zip(now, rows)]
        x = {m: rng.standard_normal((n, h, D)).astype(np.float32) for m, h in (("k", KVH), ("v", KVH), ("q", H))}
        for m, p in (("k", dk), ("v", dv), ("q", dq)):
            dev.set(p, to_type(x[m], t))
        l = 3 * rng.standard_normal((3, V)).astype(np.float32)
        dev.set(logits, l)
        dev.set(starts, np.cumsum([0] + rows).astype(np.int32))
        dev.set(lengths, np.array(now, np.int32))
        dev.set(table, c.table)
        dev.set(out, to_type(np.full((n, H, D), 7.0, np.float32), t))
        assert rt.hipGraphLaunch(gexec, stream) == 0 and rt.hipStreamSynchronize(stream) == 0
        got = from_type(dev.get(out, (n, H, D), DTYPE[t]), t)
        got_ids = dev.get(ids, (3,), np.int32)
        at = 0
        for i, r in enumerate(rows):
            to = slice(first[i] + now[i] - r, first[i] + now[i])
            c.k[to], c.v[to] = (held(rounded(x[m][at:at + r], t), kv) for m in "kv")
            at += r
        c.check(got, x["q"], rows, t, H, 50, 4, lengths=now)
        want = [plain.sample(l[i], top_p=[0.9, 1.0, 0.5][i], u=[0.1, 0.5, 0.9][i])[0] for i in range(3)]
        assert list(got_ids) == want
        step(0)
        np.testing.assert_array_equal(from_type(dev.get(out, (n, H, D), DTYPE[t]), t), got)
        np.testing.assert_array_equal(dev.get(ids, (3,), np.int32), got_ids)
    assert rt.hipGraphExecDestroy(gexec) == 0 and rt.hipGraphDestroy(graph) == 0 and rt.hipStreamDestroy(stream) == 0
    c.close()


def test_results_do_not_depend_on_the_batch_or_the_run(dev):
    """The same call twice, and beside work on another stream with a workspace of its own: the same bits."""
    c, rng = _filled(dev, "e4m3", 64, 2, 128, [900, 300, 1500])
    rows = [1, 1, 1]
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    one = c.attend(q, rows, F32, 8)
    streams = [C.c_void_p(), C.c_void_p()]
    for s in streams:
        assert dev.rt.hipStreamCreate(C.byref(s)) == 0
    b, dq = c.batch(rows), dev.put(q)
    need = c.pool.attention_workspace(b, 8, F32)
    outs, works = [dev.empty(q.nbytes) for _ in streams], [dev.empty(need) for _ in streams]
    for _ in range(10):
        for s, o, w in zip(streams, outs, works):
            c.pool.attention(0, b, dq, o, 8, F32, workspace=w, workspace_bytes=need, stream=s.value)
    for o in outs:
        np.testing.assert_array_equal(dev.get(o, q.shape, np.float32), one)
    for s in streams:
        assert dev.rt.hipStreamDestroy(s) == 0
    c.close()


def test_a_workspace_for_any_limits(dev):
    """The smallest, the largest and any limits between have a plan; empty calls want no workspace and do nothing."""
    from llama2_rs import ops
    rng = np.random.default_rng(12)
    pools = [ops.KvPool(1, 4, 64, heads, d, kv) for heads, d, kv in ((1, 64, "i8"), (8, 128, "bf16"))]
    ends = [0, 1, 2, 3, 16, 17, 64, 65, 255, 256, 257, 4096]
    any_of = lambda most: int(rng.choice(ends + [most])) if rng.random() < 0.7 else int(2 ** rng.uniform(0, np.log2(most)))  # noqa: E731
    for n in range(4000):
        p = pools[n % 2]
        seqs, rows, most, length = min(any_of(65535), 65535), min(any_of(1 << 22), 1 << 22), any_of(1 << 22), any_of(1 << 30)
        group = int(rng.choice([1, 2, 3, 8, 16, 17, 33, 64, 65, 255]))
        b = ops.KvBatch(64, 64, 64, seqs, -(-length // 64), rows, most, length)
        need = p.attention_workspace(b, group * (8 if n % 2 else 1), int(rng.integers(3)), int(rng.choice([0, 1, 100, 2 ** 31 - 1])), int(rng.choice([0, 5, 2 ** 31 - 1])))
        assert 0 <= need < 2 ** 62
        if seqs == 0 or rows == 0 or most == 0:
            p.attention(0, b, 0, 0, group * (8 if n % 2 else 1))
    for p in pools:
        p.close()


def test_contents_beyond_the_limits_touch_nothing_else(dev):
    """Arrays that say more than the call's limits: nothing outside of the rows and the pool's own pages is written."""
    c, rng = _filled(dev, "i8", 16, 1, 64, [64, 64])
    from llama2_rs import ops
    q = rng.standard_normal((12, 2, 64)).astype(np.float32)
    for starts, lengths in (([0, 5, 4000], [64, 64]), ([-7, 5, 9], [64, 1 << 30]), ([0, 9, 3], [-5, 64]), ([0, 2, 4], [1000, 2000])):
        b = ops.KvBatch(dev.put(np.array(starts, np.int32)), dev.put(np.array(lengths, np.int32)), dev.put(c.table), 2, c.max_pages, 8, 6, 64)
        got = c.attend(q, None, F32, 2, batch=b)
        assert np.all(got[8:] == 7.0)
        before = _read(c, dev, [64, 64], F32)
        out = dev.put(np.full((12, 1, 64), 7.0, np.float32))
        c.pool.read(0, b, out, out, F32)
        assert np.all(dev.get(out, (12, 1, 64), np.float32)[8:] == 7.0)
        for x, y in zip(before, _read(c, dev, [64, 64], F32)):
            np.testing.assert_array_equal(x, y)
    c.close()


def test_refusals(dev):
    from llama2_rs import ops
    from llama2_rs._lib import L2Error
    c, rng = _filled(dev, "i8", 16, 2, 64, [40])
    b, p = c.batch([1]), dev.empty(1 << 16)
    call = dict(n_heads=4, workspace=p, workspace_bytes=1 << 16)
    c.pool.attention(0, b, p, p, **call)
    for bad in (dict(n_heads=3), dict(n_heads=0), dict(window=-1), dict(sinks=-1), dict(type=3), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(q_stride=255), dict(out_stride=-256)):
        with pytest.raises(L2Error):
            c.pool.attention(0, b, p, p, **{**call, **bad})
    need = c.pool.attention_workspace(b, 4)
    for layer, q, o, more in ((1, p, p, {}), (-1, p, p, {}), (0, 0, p, {}), (0, p, 0, {}), (0, p + 2, p, {}), (0, p, p + 1, {}),
                              (0, p, p, dict(workspace=0)) if need else (1, p, p, {}), (0, p, p, dict(workspace_bytes=need - 1)) if need else (1, p, p, {}),
                              (0, p, p, dict(workspace=p + 4)) if need else (1, p, p, {})):
        with pytest.raises(L2Error):
            c.pool.attention(layer, b, q, o, **{**call, **more})
    for f in (c.pool.write, c.pool.read):
        for layer, k, v, more in ((1, p, p, {}), (0, 0, p, {}), (0, p, 0, {}), (0, p + 2, p, {}), (0, p, p, dict(type=-1)), (0, p, p, dict(k_stride=127)),
                                  (0, p, p, dict(v_stride=-1))):
            with pytest.raises(L2Error):
                f(layer, b, k, v, **more)
    for change in (dict(n_seqs=-1), dict(n_seqs=65536), dict(max_pages=2), dict(max_length=49), dict(n_rows=-1), dict(max_rows=-1), dict(starts=None),
                   dict(lengths=None), dict(pages=None), dict(n_rows=(1 << 22) + 1)):
        bb = c.batch([1])
        for name, value in change.items():
            setattr(bb, name, value)
        with pytest.raises(L2Error):
            c.pool.attention(0, bb, p, p, **call)
    # calls that have nothing to do
    for change in (dict(n_seqs=0), dict(n_rows=0), dict(max_rows=0)):
        bb = c.batch([1])
        for name, value in change.items():
            setattr(bb, name, value)
        c.pool.attention(0, bb, 0, 0, n_heads=4)
        c.pool.write(0, bb, 0, 0)
        c.pool.read(0, bb, 0, 0)
    with pytest.raises(L2Error):
        ops.KvPool(1, 1 << 30, 256, 1000, 128, "f16")
    c.close()
