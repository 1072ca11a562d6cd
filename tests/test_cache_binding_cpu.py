"""The binding of the cache calls refuses numbers that the C ABI would see cut off."""
import numpy as np
import pytest

from juno_b200.matvec import PagedKvCache


class Tensor:
    """As much of a CUDA tensor as the binding looks at."""
    is_cuda = True

    def __init__(self, shape, dtype="float32"):
        self.shape, self.dtype = shape, f"torch.{dtype}"

    def stride(self):
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


class Library:
    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was reached")
        return call


@pytest.mark.parametrize("number", [1 << 31, (1 << 32) + 1, -(1 << 31) - 1, -(1 << 32) + 1])
def test_numbers_beyond_32_bits(number):
    cache = PagedKvCache.__new__(PagedKvCache)
    cache._L, cache.ctx, cache.handle = Library(), type("Context", (), {"handle": None})(), None
    cache.n_layers, cache.n_kv_heads, cache.head_dim = 2, 2, 64
    rows, q, w = Tensor((1, 128)), Tensor((1, 256)), Tensor((1, 2, 1))
    for call in (lambda: cache.append_device(number, [None], [0], [1], rows, rows), lambda: cache.read_device(number, [None], [0], [1], rows, rows),
                 lambda: cache.attention_device(number, [None], q, 4, q), lambda: cache.weights_device(number, [None], [1], w),
                 lambda: cache.evict([None], number), lambda: cache.evict([None], 1, number), lambda: cache.fork(None, number)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
