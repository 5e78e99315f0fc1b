"""Refusals of the Python calls on 4-bit caches, and what they leave alone."""
import numpy as np
import pytest

from ratchet_amd import DType, Device, InvariantError, OperationError, Tensor, _ffi

CPU = Device.CPU


def halves(*shape):
    return Tensor.from_data(np.zeros(shape, np.float16))


@pytest.mark.parametrize("shape", [(64, 64), (4, 32, 32), (2, 3, 20, 64), (1, 1, 2, 20, 64)])
def test_a_weight_of_any_rank_is_no_cache(shape):
    w = Tensor(shape, DType.Q4_0, CPU, np.zeros(0, np.uint8))
    with pytest.raises(InvariantError) as e:
        w.cache_write(halves(2, 3, 1, 64), 0)
    assert e.value.status == _ffi.RT_ERR_DTYPE_MISMATCH
