"""The largest scales of the attention over sequences of different lengths: kernels work in base 2, so that scale * log2(e) has to be a number too."""
import ctypes
import math

import pytest
import torch

from ragged_cases import Paged, attend_packed, attend_paged, cache_desc, close, packed_desc, paged_desc, starts_of
from ratchet_amd import _ffi

gpu = pytest.mark.gpu
MOST = 2.0**127 * (2 - 2.0**-23) / math.log2(math.e)      # 2.3586e38


@pytest.mark.parametrize("scale,fine", [(0.99999 * MOST, True), (1.00001 * MOST, False), (3e38, False), (3.4e38, False), (1e38, True), (float("inf"), False), (float("nan"), False)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scales_that_are_taken(scale, fine, sign):
    need, status = ctypes.c_uint64(), _ffi.RT_OK if fine else _ffi.RT_ERR_INVALID_ARG
    L = _ffi.lib()
    d = paged_desc(cache_desc(2, 2, 64, 10, 16, 4), 8, 10, 8, 64, True, sign * scale)
    assert L.rt_attention_paged_validate(d) == status and L.rt_attention_paged_workspace_bytes(d, need) == status
    d = packed_desc(2, 8, 2, 64, 10, 10, 8, 8, True, sign * scale)
    assert L.rt_attention_packed_validate(d) == status and L.rt_attention_packed_workspace_bytes(d, need) == status


@gpu
@pytest.mark.parametrize("scale", [0.99999 * MOST, -0.99999 * MOST, 1e30])
@pytest.mark.parametrize("rows,keys", [(1, 700), (6, 90), (6, 5000), (150, 200)])
def test_scores_of_zero(device, scale, rows, keys):
    """A query of zeros weighs all keys alike, whatever the scale and the rows beside it."""
    n, d = [rows, rows], 64
    c = Paged(rows, [keys, keys + 3], 2, d, 16)
    q = torch.randn((2 * rows, 4, d), generator=torch.Generator().manual_seed(1)).half()
    q[::2] = 0
    k_pool, v_pool, table, lens = c.on_gpu()
    paged, packed = (torch.empty(q.shape, dtype=torch.float16, device="cuda") for _ in range(2))
    attend_paged(device, paged_desc(c.cache, 4, 2 * rows, rows, c.width * 16, False, scale), q.cuda(), k_pool, v_pool, table, lens, starts_of(n).cuda(), paged)
    attend_packed(device, packed_desc(2, 4, 2, d, 2 * rows, 2 * keys + 3, rows, keys + 3, False, scale), q.cuda(), torch.cat(c.k).cuda(), torch.cat(c.v).cuda(), starts_of(n).cuda(),
                  starts_of(c.lens).cuda(), packed)
    v = [x.double().repeat_interleave(2, 1) for x in c.v]
    mean, size = (torch.cat([f(x)[None].expand(rows, 4, d) for x in v]) for f in (lambda x: x.mean(0), lambda x: x.abs().mean(0)))
    # equal probabilities are rounded alike, which cancels; sums of so many terms in f32, the output's rounding
    tol = (keys + 3) * 2.0**-24 * 2 * size + 2.0**-11 * mean.abs() + 2.0**-25
    for out, what in ((paged, "paged"), (packed, "packed")):
        close(out[::2], mean[::2], tol[::2], (what, scale))
