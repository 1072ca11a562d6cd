"""4-bit cache pages on the CPU: the numbers of a group are decided exactly, the layout covers a block once, the oracle is pinned to plain formulas,
calls without a context are refused."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

from juno_b200 import _lib
from oracle import q4_cache_oracle as q4
from q4util import host_library, rows


@pytest.fixture(scope="module")
def host():
    return host_library()


@pytest.mark.parametrize("hd", [64, 128])
def test_a_block_holds_every_number_and_factor_once(host, hd):
    n = host.q4_host_block_bytes(hd)
    assert n == 16 * 2 * hd * 5 // 8
    nibbles = np.zeros(2 * n, dtype=np.uint8)
    assert host.q4_host_cover(hd, nibbles.ctypes.data_as(C.c_void_p)) == 0
    assert (nibbles == 1).all()


def test_the_numbers_of_a_unit(host):
    out = (C.c_int * 4)()
    for n in range(1 << 16):
        want = [n >> 4 * i & 15 for i in range(4)]
        host.q4_host_unit(*want, out)
        assert list(out) == want


def _nearest(x, m, d):
    """In rational numbers: the whole number nearest to (x - m) / d, ties to even, within [0, 15]."""
    return max(0, min(15, round((Fraction(float(x)) - Fraction(float(m))) / Fraction(float(d)))))


def test_numbers_are_decided_exactly(host):
    rng = np.random.default_rng(5)
    cases = []
    for _ in range(400):
        m = np.float32(np.float16(rng.standard_normal() * 10.0 ** rng.integers(-3, 3)))
        d = q4.bf16(np.float32(abs(rng.standard_normal()) * 10.0 ** rng.integers(-6, 3) + 1e-30))
        for k in range(-1, 17):
            edge = np.float32(float(m) + (k + 0.5) * float(d))  # half-way between two numbers, and the values beside it
            cases += [(v, m, d) for v in (edge, np.nextafter(edge, np.float32(np.inf)), np.nextafter(edge, np.float32(-np.inf)))]
        cases.append((np.float32(float(m) + 15.0 * rng.random() * float(d)), m, d))
    # x - m rounds to the half-way point itself here: what the rounding took away decides
    cases += [(np.float32(v), np.float32(m), np.float32(2.0)) for m in (-1.0, -3.0, -5.0) for v in (1e-30, 0.0, -1e-30)]
    for x, m, d in cases:
        assert host.q4_host_number(float(x), float(m), float(d)) == _nearest(x, m, d), (x, m, d)
        assert host.q4_host_number_exact(float(x), float(m), float(d)) == _nearest(x, m, d), (x, m, d)
    assert host.q4_host_number(3.0, 1.0, 0.0) == host.q4_host_number_exact(3.0, 1.0, 0.0) == 0


def test_oracle_numbers_agree_with_the_host_functions(host):
    rng = np.random.default_rng(6)
    x = rows(rng, 40, 2, 64)
    q, d, m = q4.quantise(x)
    g = x.reshape(40, 2, 2, 32)
    for i in np.ndindex(40, 2, 2):
        got = [host.q4_host_number(float(v), float(m[i][0]), float(d[i][0])) for v in g[i]]
        assert got == q[i].astype(int).tolist()


def test_oracle_values_lie_within_half_a_step():
    rng = np.random.default_rng(7)
    x = rows(rng, 300, 2, 128)
    q, d, m = q4.quantise(x)
    off = np.abs((m + d * q) - x.reshape(q.shape))
    # half a step; beyond the last number what the step's rounding takes off 15 steps (2^-8 of it), before the first what the offset's takes (2^-11 of it)
    assert (off <= d * (0.5 + 15 * 2.0 ** -8) + np.abs(m) * 2.0 ** -11).all()
    assert q.min() == 0 and q.max() == 15


def test_oracle_special_groups():
    x = np.zeros((1, 1, 96), dtype=np.float32)
    x[..., 3] = np.nan
    x[..., 40], x[..., 41] = np.inf, -np.inf
    x[..., 64:] = np.float32(7.25)
    v = q4.held(x)[0, 0]
    assert np.isnan(v[:32]).all()
    assert v[41] == -65504 and abs(v[40] - 65504) <= 15 * 2.0 ** -8 * 131008 / 15 and np.isfinite(v[32:64]).all()
    assert (v[64:] == 7.25).all()


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(8)
    q, k, v = rng.standard_normal((4, 32)), rng.standard_normal((9, 2, 32)), rng.standard_normal((9, 2, 32))
    out, w = q4.attention(q, k, v)
    for h in range(4):
        e = np.exp(k[:, h // 2] @ q[h] / np.sqrt(32))
        assert np.allclose(out[h], (e / e.sum()) @ v[:, h // 2], rtol=1e-12)
    assert np.allclose(w.sum(-1), 2.0)


def test_oracle_eviction():
    w = [3.0, 1.0, 1.0, np.nan, 0.0, 1.0, 9.0, 0.0]
    assert q4.kept(w, 4, 1).tolist() == [0, 1, 6, 7]
    assert q4.kept(w, 4, 0).tolist() == [0, 1, 2, 6]
    assert q4.kept(w, 7, 0).tolist() == [0, 1, 2, 4, 5, 6, 7]
    assert q4.kept(w, 3, 3).tolist() == [5, 6, 7]
    assert q4.kept(w, 8, 2).tolist() == list(range(8))


def test_calls_without_handles_are_refused():
    L = _lib.load()
    one = (C.c_void_p * 1)()
    assert L.juno_kvpool_track(None, 1, 16) == _lib.ERR_INVALID_ARG
    assert L.juno_seq_track(None) == _lib.ERR_INVALID_ARG
    assert L.juno_kv_append_device(None, None, 0, 1, one, None, None, None, None, 64, None) == _lib.ERR_INVALID_ARG
    assert L.juno_kv_read_device(None, None, 0, 1, one, None, None, None, None, 64, None) == _lib.ERR_INVALID_ARG
    assert L.juno_kv_weights_device(None, None, 0, 1, one, None, None, 16, 0, None) == _lib.ERR_INVALID_ARG
    assert L.juno_attn_decode_device(None, None, 0, 1, one, None, 8, None, 64, None, 64, None) == _lib.ERR_INVALID_ARG
    assert L.juno_kv_evict(None, None, 1, one, 16, 0, None, None) == _lib.ERR_INVALID_ARG
    assert "context is null" in _lib.last_error()


def test_binding_refuses_what_is_not_a_tensor():
    from juno_b200.matvec import PagedKvCache, _device_ptr
    with pytest.raises(ValueError, match="not a tensor"):
        _device_ptr(np.zeros((1, 4), np.float32), "q", 1, 4)
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="CUDA tensor"):
        _device_ptr(torch.zeros(1, 4), "q", 1, 4)
    with pytest.raises(ValueError, match="whole numbers"):
        PagedKvCache._ints([1, 2], 3, "counts")
    assert PagedKvCache._stream(None) is None and PagedKvCache._stream(0) == 1 and PagedKvCache._stream(77) == 77


def test_lengths_are_whole_numbers_of_32_bits():
    from juno_b200.matvec import PagedKvCache
    ints = PagedKvCache._ints
    for x in ([1, 2], (1, 2), np.array([1, 2]), np.array([1, 2], dtype=np.uint8), np.array([1, 9, 2], dtype=np.int32)[::2]):
        a = ints(x, 2, "lens")
        assert a.dtype == np.int32 and a.tolist() == [1, 2]
    for x in ([1.0, 2.0], [1], [[1, 2]], [True, False], [1, 2 ** 32 + 1], np.array([1, 2 ** 31]), ["1", "2"]):
        with pytest.raises(ValueError):
            ints(x, 2, "lens")
