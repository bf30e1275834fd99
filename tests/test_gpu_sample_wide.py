"""Sampling on the device from the most logits that it takes, and refused above."""
import numpy as np
import pytest

from tests.kvpool_plain import BF16, F32, rounded
from tests.test_gpu_sample import _ids, _logits, _u, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _answers(row, got, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Whether `got` is an answer in exact arithmetic, of weights that are each off by up to 2^-45 of the largest: a sum of n of them is off by n times that, so
    a running sum, and the border that a filter draws at one, lie within n 2^-44 (the sum and what it is compared with); tokens between the borders drawn
    that much apart may be kept or not, and what they weigh may be in the sums or not."""
    x = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return got == order[0]
    w = np.exp((x - x[order[0]]) / np.float64(np.float32(temperature)))
    tol = len(x) * 2.0 ** -44
    if 0 < top_k < len(x):
        order = order[:top_k]
    least = most = len(order)
    if top_p < 1:
        c = np.cumsum(w[order])
        target = float(np.float32(top_p)) * c[-1]
        least, most = (min(int(np.searchsorted(c, target + s * tol)) + 1, len(order)) for s in (-1, 1))
    surely = maybe = None
    for n, sign in ((least, 1), (most, -1)):
        kept = order[:n]
        if min_p > 0:
            kept = kept[(w[kept] >= min(float(np.float32(min_p)), 1.0) + sign * 2.0 ** -44) | (x[kept] == x[order[0]])]
        surely, maybe = (kept, maybe) if sign > 0 else (surely, kept)
    loose = w[maybe].sum() - w[surely].sum() + tol
    if got not in maybe:
        return False
    m = np.zeros(len(x))
    m[surely] = w[surely]
    c = np.cumsum(m)
    target = min(max(float(np.float32(u)), 0.0), 1.0) * c[-1]
    return c[got] - m[got] - 2 * loose <= target <= c[got] + 2 * loose


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("vocab", [(1 << 19) - 3, 1 << 19])
def test_the_largest_vocabulary(dev, vocab, t):  # noqa: F811
    rng = np.random.default_rng(vocab)
    x = _logits(rng, 4, vocab)
    x[1, vocab - 1] = x[1].max() + 3
    u = _u(rng, 4)
    u[2] = 1 - 2.0 ** -24
    flat = np.zeros((2, vocab), np.float32)
    flat[1, ::2] = -np.inf
    for rows, all_u, all_settings in ((x, u, ({}, dict(temperature=0.0), dict(top_k=vocab - 1), dict(top_k=1000, temperature=3.0), dict(top_p=0.95),
                                              dict(top_p=0.9999, temperature=1.5), dict(min_p=0.001), dict(top_k=5000, top_p=0.9, min_p=0.01))),
                                      (flat, _u(rng, 2), ({}, dict(top_k=vocab // 2), dict(top_p=0.25)))):
        for settings in all_settings:
            got = _ids(dev, rows, all_u, t, **{n: np.full(len(rows), a) for n, a in settings.items()})
            for i, row in enumerate(rounded(rows, t)):
                assert _answers(row, got[i], all_u[i], **settings), (i, settings, got[i])


def test_a_model_of_more_tokens_is_refused_before_its_step():
    """l2_decode_sample on a vocabulary that sampling does not take: refused, and the cache is as it was."""
    from llama2_rs import checkpoint as ck, ops
    from llama2_rs._lib import L2Error
    dims = ck.Dims(dim=128, hidden_dim=128, n_layers=1, n_heads=1, n_kv_heads=1, vocab_size=(1 << 19) + 1, seq_len=16, group_size=0)
    m = ops.Model(np.full(ck.weights_bytes(dims) // 4, 0.01, np.float32).view(np.uint8), dims)
    m.forward([1], [0])
    before = m.read_kv(0, 0, 2)
    assert before[0][0].any()
    with pytest.raises(L2Error):
        m.decode_sample(2, 1, 0.5)
    for x, y in zip(m.read_kv(0, 0, 2), before):
        np.testing.assert_array_equal(x, y)
    m.close()
