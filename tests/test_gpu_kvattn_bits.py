"""Attention over a cache in pages: how many bits its results have, and at the ends of what the types hold, against 64-bit arithmetic."""
import numpy as np
import pytest

from tests import kvpool_plain as plain
from tests.kvpool_plain import BF16, F16, F32, Cache, Device, rounded

pytestmark = pytest.mark.gpu
KV = ("i8", "e4m3", "f16", "bf16")
TINY = {F32: 2.0 ** -130, F16: 2.0 ** -25, BF16: 2.0 ** -130}


@pytest.fixture()
def dev():
    from llama2_rs import _lib
    assert _lib.lib().l2_device_count() >= 1, "no HIP device: the GPU tests cannot run"
    d = Device()
    yield d
    d.close()


def _weight(kv, t):
    """What is left of a weight by the numbers that it enters the product as: two of 11 bits; over bf16 two of 8, three for fp32 rows."""
    return 2.0 ** -22 if kv != "bf16" else 2.0 ** -24 if t == F32 else 2.0 ** -16


def _bound(kv, t, q, k, v, scale, want):
    """Element by element.  A score's products and their sum are off by a rounding each, its factors by four; the quotient by twice what the
    score is off, by its weight's numbers, the exponential (2^-22) and the n roundings of a sum; over fp16 and 8 bits a weight is known to no less than
    2^-32 of the largest (in 8 bits times the scale of its values, which is 2^-6 of the row's largest or less)."""
    n, D = v.shape
    most = float((np.abs(k.astype(np.float64)) @ np.abs(q.astype(np.float64))).max() * scale)
    score = most * ((D + 4) * 2.0 ** -24 + (2.0 ** -21 if t == F32 else 0.0))
    s = k.astype(np.float64) @ q.astype(np.float64) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    size = p @ np.abs(v.astype(np.float64))
    off = size * (2 * score + _weight(kv, t) + 2.0 ** -21 + (n + 64) * 2.0 ** -24)
    if kv == "f16":
        off = off + 2.0 ** -32 * p.max() * np.abs(v).sum(0)
    elif kv != "bf16":
        a = np.maximum(np.abs(v).max(1), 2.0 ** -60).astype(np.float64)
        off = off + 2.0 ** -32 * (p * a).max() * (np.abs(v) / a[:, None]).sum(0)
    return 1.01 * off + (np.abs(want) + off) * plain.HALF_STEP[t] + TINY[t]


def _check(c, kv, t, got, q, rows, heads, scale=None, lengths=None):
    """Every row of `got`, all of which see all positions up to their own; NaN and infinities where the formula has them."""
    scale = c.head_size ** -0.5 if scale is None else scale
    q, at = rounded(q, t), 0
    for i, n in enumerate(rows):
        k, v = c.k[c.rows_of(i)], c.v[c.rows_of(i)]
        for j in range(n):
            upto = c.lengths[i] - n + j + 1
            for h in range(heads):
                kk, vv, g = k[:upto, h // (heads // c.kv_heads)], v[:upto, h // (heads // c.kv_heads)], got[at, h]
                want = plain.attention_row(q[at, h], kk, vv, scale)[0]
                fine = np.isfinite(vv).all(0)
                where = f"sequence {i} row {j} head {h}"
                assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isinf(g), np.isinf(want)), where
                np.testing.assert_array_equal(g[~np.isfinite(want)], want[~np.isfinite(want)].astype(np.float32))
                if np.isnan(want).all():
                    continue
                bound = _bound(kv, t, q[at, h], kk, vv[:, fine], scale, want[fine])
                off = np.abs(g[fine].astype(np.float64) - want[fine])
                assert np.all(off <= bound), (where, float(np.max(off / bound)))
            at += 1


def _cache(dev, kv, t, lengths, k=None, v=None, seed=0, head_size=64):
    c = Cache(dev, kv, 16, 1, head_size, lengths, seed=seed)
    rng = np.random.default_rng(seed + 1)
    shape = (sum(lengths), 1, head_size)
    k = rng.standard_normal(shape).astype(np.float32) if k is None else k
    v = rng.standard_normal(shape).astype(np.float32) if v is None else v
    c.fill(k, v, t)
    return c, rng


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,rows", [([5, 12, 40, 23], [1, 3, 16, 2]), ([100], [100])])
@pytest.mark.parametrize("head_size", [64, 128])
def test_weights_have_more_bits_than_results(dev, kv, t, lengths, rows, head_size):
    """Few positions with weights much alike: what a result is off by is its own rounding, and next to nothing of the weights'."""
    c, rng = _cache(dev, kv, t, lengths, head_size=head_size)
    q = (0.02 * rng.standard_normal((sum(rows), 2, head_size))).astype(np.float32)
    _check(c, kv, t, c.attend(q, rows, t, 2), q, rows, 2)
    c.close()


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("lengths,rows", [([2, 90, 200], [1, 2, 3]), ([150], [100])])
@pytest.mark.parametrize("ratio", [0, 10, 17, 24, 45])
def test_large_values_of_next_to_no_weight(dev, kv, t, lengths, rows, ratio):
    """Values 2^ratio times the others', of rows whose weight is e^-50 of the others': those keep their bits."""
    rng = np.random.default_rng(ratio)
    n, D = sum(lengths), 64
    ratio = min(ratio, 13) if t == F16 else ratio
    k, v = np.zeros((n, 1, D), np.float32), rng.standard_normal((n, 1, D)).astype(np.float32)
    large = np.zeros(n, bool)
    at = 0
    for m in lengths:
        large[[at + x for x in (0, 40, 41, 64, 100) if x < m]] = True
        at += m
    k[:, 0, 1] = 0.01 * rng.standard_normal(n)
    k[large, 0, 0] = -50
    v[large] *= np.float32(2.0 ** ratio)
    c, _ = _cache(dev, kv, t, lengths, k, v)
    q = np.zeros((sum(rows), 2, D), np.float32)
    q[..., 0], q[..., 1] = 8, rng.standard_normal((sum(rows), 2))
    _check(c, kv, t, c.attend(q, rows, t, 2), q, rows, 2)
    c.close()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t,size,scale", [(F32, 1e-41, None), (F32, 2.0 ** -149, None), (F32, 1e-12, 1e-30), (F32, 1e-38, 1e-38), (BF16, 2.0 ** -133, 1e-6),
                                          (BF16, 1e-38, None), (F16, 2.0 ** -24, 1e-36), (F32, 2.0 ** 100, 2.0 ** -100), (F32, 1e-20, 1e-44)])
@pytest.mark.parametrize("lengths,rows", [([5, 90, 37], [1, 3, 2]), ([130], [100])])
def test_factors_at_the_ends_of_fp32(dev, kv, t, size, scale, lengths, rows):
    """Queries and scales whose product is next to nothing, or which lie far apart: what is not seen stays out, and scores are what they are."""
    c, rng = _cache(dev, kv, t, lengths)
    q = (size * np.sign(rng.standard_normal((sum(rows), 2, 64)))).astype(np.float32)
    scale = None if scale is None else float(np.float32(scale))
    got = c.attend(q, rows, t, 2, scale=scale or 0.0)
    assert np.isfinite(got).all()
    _check(c, kv, t, got, q, rows, 2, scale)
    c.close()


@pytest.mark.parametrize("kv", ["i8", "e4m3", "bf16"])
@pytest.mark.parametrize("lengths,rows", [([5, 90, 37], [1, 3, 2]), ([130], [100])])
def test_keys_of_1e33(dev, kv, lengths, rows):
    """Large keys and small queries: scores are small, whatever the sums before the factors are."""
    rng = np.random.default_rng(3)
    k = (2.0 ** 110 * rng.standard_normal((sum(lengths), 1, 64))).astype(np.float32)
    c, _ = _cache(dev, kv, F32, lengths, k)
    q = (2.0 ** -111 * rng.standard_normal((sum(rows), 2, 64))).astype(np.float32)
    _check(c, kv, F32, c.attend(q, rows, F32, 2), q, rows, 2)
    c.close()


@pytest.mark.parametrize("kv", ["f16", "bf16"])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,rows", [([1500], [1]), ([70, 400], [3, 2]), ([300], [100])])
def test_infinite_values_that_are_seen(dev, kv, t, lengths, rows):
    """An infinity in a dimension of values makes the result that, and NaN NaN, whatever its weight and how many rows see its tile; both infinities are NaN; other dimensions
    are as they were."""
    rng = np.random.default_rng(5)
    n = sum(lengths)
    k, v = (rng.standard_normal((n, 1, 64)).astype(np.float32) for _ in "kv")
    inf = np.inf
    v[2, 0, 5], v[3, 0, 6], v[9, 0, 6], v[20, 0, 7], v[21, 0, 8], v[40, 0, 9], v[40, 0, 63] = inf, -inf, inf, -inf, np.nan, inf, -inf
    v[n - 20, 0, 10], v[n - 1, 0, 11] = -inf, inf
    k[20, 0], k[40, 0] = -20, 20
    c, _ = _cache(dev, kv, t, lengths, k, v)
    q = rng.standard_normal((sum(rows), 2, 64)).astype(np.float32)
    q[:, 0] = 1  # the keys of 20 and 40 decide nearly alone
    _check(c, kv, t, c.attend(q, rows, t, 2), q, rows, 2)
    c.close()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("lengths,rows", [([5, 90, 37], [1, 3, 2]), ([130], [100])])
def test_values_of_1e36_in_bf16(dev, t, lengths, rows):
    """The sum of weights times values stays finite where their mean is."""
    rng = np.random.default_rng(6)
    v = (2.0 ** 117 * rng.standard_normal((sum(lengths), 1, 64))).astype(np.float32)
    c, _ = _cache(dev, "bf16", t, lengths, None, v)
    q = rng.standard_normal((sum(rows), 2, 64)).astype(np.float32)
    _check(c, "bf16", t, c.attend(q, rows, t, 2), q, rows, 2)
    c.close()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("lengths,rows", [([1500, 300], [1, 3]), ([700], [100])])
def test_the_largest_values_of_bf16(dev, t, lengths, rows):
    """Values of one sign near the type's largest: their mean is one of them, though a sum of two is none."""
    rng = np.random.default_rng(8)
    v = (3e38 * (1 - 0.1 * rng.random((sum(lengths), 1, 64)))).astype(np.float32)
    c, _ = _cache(dev, "bf16", t, lengths, None, v)
    q = (0.01 * rng.standard_normal((sum(rows), 2, 64))).astype(np.float32)  # weights much alike
    _check(c, "bf16", t, c.attend(q, rows, t, 2), q, rows, 2)
    c.close()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,rows", [([700], [1]), ([70, 150], [20, 3]), ([150], [100])])
def test_keys_and_queries_that_are_not_finite(dev, kv, t, lengths, rows):
    """NaN in a key or a query makes every row NaN that sees it, or is it, and no other; an infinity no number where the formula has none."""
    rng = np.random.default_rng(7)
    n = sum(lengths)
    k = rng.standard_normal((n, 1, 64)).astype(np.float32)
    k[n - 2, 0, 3] = np.nan
    if len(lengths) > 1:
        k[lengths[0] - 5, 0, 4] = np.inf
    c, _ = _cache(dev, kv, t, lengths, k)
    q = rng.standard_normal((sum(rows), 2, 64)).astype(np.float32)
    q[0, 1, 9] = np.nan
    got = c.attend(q, rows, t, 2)
    at = 0
    for i, m in enumerate(rows):
        for j in range(m):
            upto = lengths[i] - m + j + 1
            kk, vv = c.k[c.rows_of(i)][:upto, 0], c.v[c.rows_of(i)][:upto, 0]
            for h in range(2):
                qq = rounded(q[at, h], t)
                if np.isnan(kk).any() or np.isnan(qq).any():
                    assert np.isnan(got[at, h]).all(), (i, j, h)
                elif not np.isfinite(kk).all():
                    want = plain.attention_row(qq, kk, vv, 0.125)[0]
                    assert np.isnan(got[at, h]).all() or np.isfinite(want).all(), (i, j, h)
                else:
                    want = plain.attention_row(qq, kk, vv, 0.125)[0]
                    assert np.all(np.abs(got[at, h] - want) <= _bound(kv, t, qq, kk, vv, 0.125, want)), (i, j, h)
            at += 1
    c.close()
