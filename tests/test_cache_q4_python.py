"""Refusals of the Python calls on 4-bit caches, and what they leave alone."""
import numpy as np
import pytest

from ratchet_amd import DType, Device, InvariantError, OperationError, Tensor, _ffi, nn
from ratchet_amd.tensor import cache_q4_nbytes

CPU = Device.CPU


def halves(*shape):
    return Tensor.from_data(np.zeros(shape, np.float16))


@pytest.mark.parametrize("shape", [(64, 64), (4, 32, 32), (2, 3, 20, 64), (1, 1, 2, 20, 64)])
def test_a_weight_of_any_rank_is_no_cache(shape):
    w = Tensor(shape, DType.Q4_0, CPU, np.zeros(0, np.uint8))
    with pytest.raises(InvariantError) as e:
        w.cache_write(halves(2, 3, 1, 64), 0)
    assert e.value.status == _ffi.RT_ERR_DTYPE_MISMATCH


def test_sizes_past_31_bits():
    """What does not fit the interface's int32 is refused, not taken modulo 2^32: a cache of 2^32 + 5 rows had the bytes of one of 5, and a write at row 2^32 + 1 went to row 1."""
    for shape in ((1, 1, 2**32 + 5, 64), (2**32 + 1, 1, 8, 64), (1, 2**32 + 1, 8, 64), (1, 1, 8, 2**32 + 64), (1, 1, 2**31, 64), (1, 1, -1, 64)):
        with pytest.raises(OperationError) as e:
            Tensor.empty_cache(shape, CPU, DType.Q4_0)
        assert e.value.status == _ffi.RT_ERR_INVALID_SHAPE, shape
    assert cache_q4_nbytes((1, 1, 2**31 - 1, 64)) == (2**31 * 36, 2**31 * 32)


def test_types_of_a_cache():
    """F16, F32 and Q4_0; others are refused with the library's error, also through the modules."""
    for dt in (DType.F16, DType.F32):
        c = Tensor.empty_cache((1, 2, 8, 64), CPU, dt)
        assert c.dt == dt and not c.is_q4_cache and not c.storage.any()
    for make in (lambda dt: Tensor.empty_cache((1, 2, 8, 64), CPU, dt), lambda dt: nn.KVCache(1, (1, 2, 8, 64), CPU, dt)):
        for dt in (DType.Q8_0H, DType.Q8_0F, DType.Q4_K):
            with pytest.raises(OperationError) as e:
                make(dt)
            assert e.value.status == _ffi.RT_ERR_UNSUPPORTED
