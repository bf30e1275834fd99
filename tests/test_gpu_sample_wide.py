"""Sampling on the device from the most logits that it takes, and refused above."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


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
