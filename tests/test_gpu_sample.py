"""Sampling on the device against 64-bit arithmetic: the very id, except where the random number lies on a border."""
import ctypes as C

import numpy as np
import pytest

from tests import kvpool_plain as plain
from tests.kvpool_plain import BF16, F16, F32, Device, rounded, to_type

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dev():
    from llama2_rs import _lib
    assert _lib.lib().l2_device_count() >= 1, "no HIP device: the GPU tests cannot run"
    d = Device()
    yield d
    d.close()


def _ids(dev, x, u, t=F32, stride=0, offset=0, **settings):
    """One id per row of x [rows][vocab]."""
    from llama2_rs import ops
    rows, vocab = x.shape
    if stride:
        wide = np.full((rows, stride), 1e30 if t == F32 else 6e4, np.float32)  # would win if it were read
        wide[:, :vocab] = x
        flat = np.concatenate([np.full(offset, 6e4, np.float32), wide.reshape(-1)])
    else:
        flat = np.concatenate([np.full(offset, 6e4, np.float32), x.reshape(-1)])
    p = dev.put(to_type(flat, t)) + offset * plain.BYTES[t]
    ids = dev.put(np.full(rows + 1, -77, np.int32))
    of = {n: dev.put(np.asarray(a, np.int32 if n == "top_k" else np.float32)) for n, a in settings.items()}
    ops.sample_device(p, rows, vocab, ids, dev.put(np.asarray(u, np.float32)), type=t, stride=stride, **of)
    got = dev.get(ids, (rows + 1,), np.int32)
    assert got[-1] == -77
    return got[:-1]


def _check(dev, x, u, t=F32, **more):
    settings = {n: np.broadcast_to(np.asarray(a), (len(x),)) for n, a in more.items() if n not in ("stride", "offset")}
    got = _ids(dev, x, u, t, **{n: a for n, a in more.items() if n in ("stride", "offset")}, **settings)
    r = rounded(x, t)
    on_border = 0
    for i in range(len(x)):
        want, near = plain.sample(r[i], u=u[i], **{n: a[i].item() for n, a in settings.items()})
        # weights are off by 2^-45 of the largest, each, and their sum by as many of these as there are tokens
        if near < x.shape[1] * 2.0 ** -43:
            on_border += 1
            continue
        assert got[i] == want, (i, {n: a[i] for n, a in settings.items()}, u[i], near)
    assert on_border <= len(x) // 8 + 1
    return got


def _logits(rng, rows, vocab, sigma=2.0):
    x = sigma * rng.standard_normal((rows, vocab))
    for _ in range(min(vocab, 20)):
        x[np.arange(rows), rng.integers(0, vocab, rows)] += 8 * rng.random(rows)
    return x.astype(np.float32)


def _u(rng, n):
    return (rng.integers(0, 1 << 24, n) / float(1 << 24)).astype(np.float32)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 257, 1000, 4095, 4097, 32000, 32768, 32769, 50001, 131072])
def test_ids(dev, vocab, t):
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 40000 else 8
    x = _logits(rng, rows, vocab)
    for settings in ({}, dict(temperature=0.7), dict(temperature=0.0), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=1), dict(top_p=0.0),
                     dict(top_k=vocab - 1, top_p=0.999, temperature=1.5), dict(top_k=300, top_p=0.5, min_p=0.01, temperature=2.0),
                     dict(top_k=5, min_p=1.0)):
        _check(dev, x, _u(rng, rows), t, **settings)


def test_settings_of_each_row(dev):
    rng = np.random.default_rng(2)
    rows = 300
    x = _logits(rng, rows, 3001, 3.0)
    x[5], x[6], x[7, 10:] = -np.inf, np.nan, -np.inf
    got = _check(dev, x, _u(rng, rows), temperature=rng.choice([0.0, -1.0, 0.01, 0.5, 1.0, 3.0, 100.0, np.nan], rows), top_k=rng.choice([-3, 0, 1, 2, 17, 900, 3001, 1 << 30], rows),
                 top_p=rng.choice([-1.0, 0.0, 0.3, 0.9, 1.0, 2.0, np.nan], rows), min_p=rng.choice([-1.0, 0.0, 0.1, 0.9, 1.0, 7.0, np.nan], rows))
    assert got[5] == -1 and got[6] == -1 and 0 <= got[7] < 10


@pytest.mark.parametrize("vocab", [100, 5000, 40000])
def test_ties(dev, vocab):
    """Equal logits: the lower id first, in every filter; all equal, a few levels, and rows of one value but for some."""
    rng = np.random.default_rng(vocab)
    rows = 12
    for x in (np.zeros((rows, vocab)), rng.integers(0, 3, (rows, vocab)).astype(float), np.where(rng.random((rows, vocab)) < 0.001, 4.0, 1.0),
              np.where(rng.random((rows, vocab)) < 0.5, 0.0, -0.0), 1000.0 + rng.integers(0, 2, (rows, vocab)) * 1e-4):
        x = x.astype(np.float32)
        for settings in ({}, dict(temperature=0.0), dict(top_k=37), dict(top_k=vocab // 2), dict(top_p=0.25), dict(top_k=vocab // 3, top_p=0.501), dict(min_p=0.5)):
            _check(dev, x, _u(rng, rows), **settings)


def test_infinities_and_extremes(dev):
    rng = np.random.default_rng(4)
    x = _logits(rng, 16, 700)
    x[0, 5] = np.inf
    x[1, [9, 30, 400]] = np.inf
    x[2, ::2] = -np.inf
    x[3, 100:] = np.nan
    x[4] = -np.inf
    x[4, 699] = -3e38
    x[5] = np.linspace(-3e38, 3e38, 700)
    x[6] = np.linspace(-1e-40, 1e-40, 700)
    x[7] = 3.4e38
    x[8] *= 1e30
    x[9, :] = -np.inf
    for settings in ({}, dict(top_k=2), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=1e-38), dict(temperature=1e30), dict(top_k=650, top_p=0.99)):
        got = _check(dev, x, _u(rng, 16), **settings)
        assert got[0] == 5 and got[1] in (9, 30, 400) and got[4] == 699 and got[9] == -1 and got[2] % 2 == 1 and got[3] < 100


def test_random_numbers_at_the_ends(dev):
    rng = np.random.default_rng(5)
    x = _logits(rng, 8, 3000)
    u = np.array([0.0, 1.0, 1.5, -1.0, np.nan, 1 - 2.0 ** -24, 2.0 ** -30, np.inf], np.float32)
    for settings in ({}, dict(top_k=3), dict(top_p=0.5)):
        got = _ids(dev, x, u, **{n: np.broadcast_to(np.asarray(a), (8,)) for n, a in settings.items()})
        for i in range(8):
            w = 0.0 if not u[i] > 0 else min(float(u[i]), 1.0)
            assert got[i] == plain.sample(x[i], u=w, **settings)[0], (i, settings)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_strides_and_addresses(dev, t):
    rng = np.random.default_rng(6)
    x = _logits(rng, 9, 1003)
    for stride, offset in ((1003, 1), (1011, 3), (2000, 2), (1004, 0)):
        _check(dev, x, _u(rng, 9), t, stride=stride, offset=offset, top_k=100, top_p=0.9)


def test_a_row_is_the_same_in_every_batch(dev):
    rng = np.random.default_rng(7)
    x = _logits(rng, 64, 9000)
    u = _u(rng, 64)
    all_rows = _ids(dev, x, u, top_p=np.full(64, 0.9))
    for i in (0, 17, 63):
        assert _ids(dev, x[i:i + 1], u[i:i + 1], top_p=[0.9])[0] == all_rows[i]
    for _ in range(3):
        np.testing.assert_array_equal(_ids(dev, x, u, top_p=np.full(64, 0.9)), all_rows)


def test_shares(dev):
    """Evenly spaced random numbers give each token its share of them, to within one."""
    n = 4000
    x = np.tile(np.log(np.array([0.5, 0.25, 0.15, 0.07, 0.03])).astype(np.float32), (n, 1))
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = np.bincount(_ids(dev, x, u), minlength=5)
    assert np.all(np.abs(got - n * np.array([0.5, 0.25, 0.15, 0.07, 0.03])) <= 1), got


def test_decode_sample(dev):
    """A step of a model that samples on the device: the id that the step's logits give, and the cache as l2_forward leaves it."""
    from llama2_rs import checkpoint as ck, ops
    dims = ck.Dims(dim=512, hidden_dim=768, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=1000, seq_len=64, group_size=64)
    img = ck.synth_weights_image(dims, seed=3)
    a, b = ops.Model(img, dims), ops.Model(img, dims)
    rng = np.random.default_rng(0)
    token = 1
    for pos in range(12):
        settings = dict(temperature=[1.0, 30.0, 0.0][pos % 3], top_k=[0, 50][pos % 2], top_p=[1.0, 0.8][pos // 2 % 2], min_p=[0.0, 0.3][pos // 4 % 2])
        u = float(np.float32(rng.random()))
        logits = b.forward([token], [pos])
        want, near = plain.sample(logits, u=u, **settings)
        got = a.decode_sample(token, pos, u, **settings)
        assert got == want or near < 1e-9, (pos, settings)
        for x, y in zip(a.read_kv(1, 0, pos + 1), b.read_kv(1, 0, pos + 1)):
            np.testing.assert_array_equal(x, y)
        token = want
    from llama2_rs._lib import L2Error
    for bad in ((-1, 0), (1000, 0), (0, 64), (0, -1)):
        with pytest.raises(L2Error):
            a.decode_sample(*bad, 0.5)
    a.close()
    b.close()


def test_refusals(dev):
    from llama2_rs import ops
    from llama2_rs._lib import L2Error
    p = dev.empty(4096)
    good = dict(logits=p, rows=1, vocab=10, ids=p + 2048, u=p + 1024)
    dev.set(p, np.zeros(1024, np.float32))
    ops.sample_device(**good)
    for bad in (dict(logits=0), dict(ids=0), dict(u=0), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 19) + 1), dict(type=3), dict(stride=9), dict(stride=-10),
                dict(logits=p + 2)):
        with pytest.raises(L2Error):
            ops.sample_device(**{**good, **bad})
    ops.sample_device(**{**good, "rows": 0, "logits": 0})
