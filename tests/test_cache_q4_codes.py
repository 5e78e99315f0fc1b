"""Every quotient that the write of a 4-bit cache can meet: the codes come from a product with a reciprocal and have to be those of the exact quotient."""
import ctypes

import numpy as np
import pytest
import torch

from ratchet_amd import _ffi
from ratchet_amd.tensor import cache_q4_nbytes
from test_cache_q4 import held, packed

pytestmark = pytest.mark.gpu


def check(device, blocks):
    """Blocks [n, 32] of f16 as rows of one head."""
    n = len(blocks)
    shape = (1, 1, n, 32)
    src = torch.from_numpy(blocks).to("cuda:0")
    cache = torch.zeros(cache_q4_nbytes(shape)[0], dtype=torch.uint8, device="cuda:0")
    assert _ffi.lib().rt_cache_write_q4_enqueue(device.ctx, _ffi.RT_F16, cache.data_ptr(), src.data_ptr(), None, None, (ctypes.c_int64 * 3)(32 * n, 32 * n, 32), None, None, None, 1, 1,
                                                n, 0, n, 32, torch.cuda.current_stream().cuda_stream) == 0
    codes, ds, _ = held(blocks.reshape(shape))
    at = cache_q4_nbytes(shape)[1]
    got = cache.cpu().numpy()
    assert np.array_equal(got[: n * 16], packed(codes).reshape(-1))
    assert np.array_equal(got[at : at + 2 * n].view(np.float16), ds.reshape(-1))


def blocks_of(m, xs):
    """Blocks that start with m and hold all of xs."""
    xs = np.concatenate([xs, np.repeat(xs[:1], -len(xs) % 31)]).reshape(-1, 31)
    return np.concatenate([np.full((len(xs), 1), m), xs], 1)


@pytest.mark.parametrize("sign", [1, -1])
def test_an_octave_of_scales(device, sign):
    """Scales between 2^-3 and 2^-2, the largest m of each, and all x from a thirty-second of m (a quotient of a quarter) to m: other octaves are the same by powers of two."""
    m = np.arange(1024, 2048) / 1024
    _, ds, _ = held(np.repeat(m[:, None], 32, 1).astype(np.float16))
    last = np.flatnonzero(np.diff(ds[:, 0].astype(np.float64), append=0) != 0)
    assert len(last) == 129  # (the last of them rounds up to 2^-2)
    x = (np.arange(1024, 2048)[None, :] * np.exp2(np.arange(-16, -9))[:, None]).reshape(-1)
    out = []
    for i in last:
        near = x[(x >= m[i] / 32) & (x <= m[i])]
        out.append(blocks_of(sign * m[i], np.concatenate([near, -near])))
    check(device, np.concatenate(out).astype(np.float16))


@pytest.mark.parametrize("sign", [1, -1])
def test_scales_of_few_bits_and_the_limit(device, sign):
    """Magnitudes below 2^-14, whole multiples of 2^-24 as their scales are, against all smaller ones; and the last eight numbers, whose scale is the limit's."""
    out = []
    for m in list(range(1, 300)) + list(range(300, 1024, 7)):
        x = np.arange(m + 1)
        out.append(blocks_of(sign * m, np.concatenate([x, -x])) * 2.0**-24)
    for m in np.arange(2040, 2048) * 32.0:
        x = (np.arange(1024, 2048)[None, :] * np.exp2(np.arange(0, 6))[:, None]).reshape(-1)
        x = x[x <= m]
        out.append(blocks_of(sign * m, np.concatenate([x, -x])))
    check(device, np.concatenate(out).astype(np.float16))
