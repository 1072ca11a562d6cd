"""Calls on 4-bit cache pages in the forms that one operator's tests do not have: from host memory, beyond usual sizes, after failures, with pages shared in part."""
import numpy as np
import pytest

from juno_b200.matvec import PagedKvCache
from oracle import q4_cache_oracle as q4
from q4util import rows
from test_q4_cache_gpu import check_attention, check_weights, f32, fill, weights

pytestmark = pytest.mark.gpu


def test_host_attention_names_a_sequence_with_weights_once(ctx):
    rng = np.random.default_rng(51)
    cache = PagedKvCache(ctx, 1, 2, 64, 16, "q4", track_seqs=1, track_tokens=64)
    a, b = cache.new_sequence(64, track=True), cache.new_sequence(64)
    k, v = rows(rng, 40, 2, 64), f32(rng.standard_normal((40, 2, 64)))
    fill(cache, 0, [a, b], [0, 0], [(k, v)] * 2)
    q = f32(rng.standard_normal((3, 8, 64)))
    for seqs in ([a, a], [b, a, a]):
        with pytest.raises(ValueError, match="there twice"):
            cache.attention(0, seqs, q[:len(seqs)].reshape(len(seqs), -1), 8)
    assert (weights(cache, 0, [a], [40]) == 0).all()  # a refused call adds nothing
    out = cache.attention(0, [b, a, b], q.reshape(3, -1), 8).reshape(q.shape)  # without weights a sequence may be there several times
    for i in range(3):
        w = check_attention(out[i], q[i], q4.held(k), q4.held(v))
        if i == 1:
            check_weights(weights(cache, 0, [a], [40])[0], w, q[i], k)
    cache.close()
