"""rt_attention_packed_enqueue: packed sequences of different lengths against the operator in 64 bits (ragged_cases has the tolerance)."""
import ctypes
import math

import pytest
import torch

from ragged_cases import attend_packed, close, packed_desc, reference, starts_of
from ratchet_amd import _ffi

gpu = pytest.mark.gpu


def inputs(seed, rows, kv_rows, heads, kv_heads, head_dim, sharp=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = (sharp * torch.randn((rows, heads, head_dim), generator=gen)).half()
    k, v = (torch.randn((kv_rows, kv_heads, head_dim), generator=gen).half() for _ in range(2))
    return q, k, v


def split(x, sizes):
    return list(torch.split(x, list(sizes)))


def run(device, seed, n, heads, kv_heads, head_dim, causal, lens=None, scale=None, sharp=1.0, workspace=True):
    """One call against the reference; the rows behind the last sequence stay as they were."""
    keys = n if lens is None else lens
    scale = 1 / math.sqrt(head_dim) if scale is None else scale
    q, k, v = inputs(seed, sum(n) + 3, sum(keys) + (3 if lens is None else 0), heads, kv_heads, head_dim, sharp)
    want, tol = reference(q[: sum(n)], split(k[: sum(keys)], keys), split(v[: sum(keys)], keys), n, keys, scale, causal)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    d = packed_desc(len(n), heads, kv_heads, head_dim, q.shape[0], k.shape[0], max(n), max(keys), causal, scale)
    attend_packed(device, d, q.cuda(), k.cuda(), v.cuda(), starts_of(n).cuda(), None if lens is None else starts_of(lens).cuda(), out, workspace)
    close(out[: sum(n)], want, tol, (n, keys, heads, kv_heads, head_dim, causal))
    assert bool((out[sum(n):] == 7.0).all())
    return out


@gpu
@pytest.mark.parametrize("head_dim", [8, 16, 24, 40, 56, 64, 72, 80, 96, 104, 112, 120, 128])
def test_head_sizes(device, head_dim):
    run(device, head_dim, [70, 1, 133], 4, 2, head_dim, True)
    run(device, head_dim, [66, 3], 2, 2, head_dim, False)


@gpu
@pytest.mark.parametrize("n", [[1], [0, 1, 0], [2, 31, 32, 33], [63, 64, 65], [127, 128, 129], [300, 0, 5, 257], [1] * 70, [5] * 300], ids=lambda n: f"{len(n)}x{max(n)}")
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(device, n, causal):
    run(device, len(n), n, 2, 1, 64, causal)


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (6, 2), (5, 5), (20, 4), (16, 8)])
def test_shared_heads(device, heads, kv_heads):
    run(device, heads, [150, 17, 64], heads, kv_heads, 128, True)


@gpu
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_other_lengths(device, causal):
    """More and fewer keys than queries: with the causal flag the first rows of the latter see none and are NaN; a sequence without keys."""
    run(device, 3, [40, 130, 3, 64], 4, 2, 80, causal, lens=[200, 100, 0, 64])


@gpu
@pytest.mark.parametrize("head_dim,workspace", [(64, True), (128, True), (96, True), (96, False)])
def test_few_tiles_share_their_keys(device, head_dim, workspace):
    """Few rows against many keys: the keys of a tile are shared among workgroups where there is a workspace."""
    run(device, 5, [9, 40], 2, 1, head_dim, True, lens=[2500, 1111], workspace=workspace)
    run(device, 6, [64], 1, 1, head_dim, False, lens=[4001], workspace=workspace)


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0, 1e-6, 1e-30])
def test_scales(device, scale):
    run(device, 7, [90, 70], 2, 2, 64, True, scale=scale)


@gpu
@pytest.mark.parametrize("sharp", [30.0, 400.0, 4000.0])
def test_large_scores(device, sharp):
    """Scores into the hundreds of thousands: the row's weight goes to one key or to a few, and equal keys weigh the same."""
    run(device, 8, [200, 65], 2, 2, 128, True, sharp=sharp)


@gpu
@pytest.mark.parametrize("size", [1.0, 100.0, 60000.0])
def test_equal_keys_weigh_the_same(device, size):
    """All keys alike, scores up to 2^39: a row is the mean of the values, wherever its blocks lie."""
    n, heads, d = 517, 2, 128
    q, k = (torch.full((n, heads, d), size, dtype=torch.float16) for _ in range(2))
    v = torch.randn((n, heads, d), generator=torch.Generator().manual_seed(0)).half()
    for causal in (True, False):
        out = torch.empty((n, heads, d), dtype=torch.float16, device="cuda")
        attend_packed(device, packed_desc(1, heads, heads, d, n, n, n, n, causal, 1.0), q.cuda(), k.cuda(), v.cuda(), starts_of([n]).cuda(), None, out)
        mean = v.double().cumsum(0) / torch.arange(1, n + 1)[:, None, None] if causal else v.double().mean(0, keepdim=True).expand(n, heads, d)
        size_of = v.double().abs().cumsum(0) / torch.arange(1, n + 1)[:, None, None] if causal else v.double().abs().mean(0, keepdim=True).expand(n, heads, d)
        # equal probabilities are rounded alike, which cancels; sums of n terms in f32, the output's rounding
        close(out, mean, n * 2.0**-24 * 2 * size_of + 2.0**-11 * mean.abs() + 2.0**-25, (size, causal))


@gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_hidden_keys_have_no_effect(device, head_dim):
    """NaN and infinities in keys and values that rows do not see; the rows that see such a value are not finite in its dimension."""
    n, heads = [100, 150], 2
    q, k, v = inputs(9, 250, 250, heads, heads, head_dim)
    k[80], v[80] = float("nan"), float("nan")                            # the first sequence's row 80
    v[100 + 70, 0, 3], v[100 + 90, 1, 5] = float("inf"), float("-inf")   # the second's
    v[100 + 100, 1, 5] = float("inf")
    v[100 + 120, 0, 7] = float("nan")
    want, tol = reference(q, split(k, n), split(v, n), n, n, 0.1, True)
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    attend_packed(device, packed_desc(2, heads, heads, head_dim, 250, 250, 150, 150, True, 0.1), q.cuda(), k.cuda(), v.cuda(), starts_of(n).cuda(), None, out)
    got = out.double().cpu()
    odd = torch.zeros(q.shape, dtype=torch.bool)
    odd[80:100] = True
    odd[100 + 70:, 0, 3], odd[100 + 90:, 1, 5], odd[100 + 120:, 0, 7] = True, True, True
    assert not bool(torch.isfinite(got[odd]).any())
    close(torch.where(odd, want, got), want, tol)


@gpu
def test_parts_of_a_fused_projection_and_strided_outputs(device):
    heads, kv, d, n = 6, 2, 80, [33, 1, 90]
    rows = sum(n)
    gen = torch.Generator().manual_seed(1)
    qkv = torch.randn((rows, heads + 2 * kv, d), generator=gen).half()
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    want, tol = reference(q, split(k, n), split(v, n), n, n, 0.11, True)
    x, out = qkv.cuda(), torch.full((heads, rows, d + 9), 7.0, dtype=torch.float16, device="cuda")
    w = (heads + 2 * kv) * d
    desc = packed_desc(3, heads, kv, d, rows, rows, max(n), max(n), True, 0.11, [w, d], [w, d], [w, d], [d + 9, rows * (d + 9)])   # rows of outputs start anywhere
    attend_packed(device, desc, x, x[:, heads:], x[:, heads + kv:], starts_of(n).cuda(), None, out[:, :, 1:])
    close(out[:, :, 1:d + 1].transpose(0, 1), want, tol)
    assert bool((out[:, :, 0] == 7.0).all()) and bool((out[:, :, d + 1:] == 7.0).all())


@gpu
def test_rows_far_apart(device):
    """The largest strides of keys and values: rows 32 MiB apart, offsets past 2^32 within a sequence."""
    rows, d, far = 200, 64, 1 << 24
    q, k, v = inputs(14, rows, rows, 2, 1, d)
    room = torch.empty((rows - 1) * far + 2 * d, dtype=torch.float16, device="cuda")
    kv = torch.as_strided(room, (rows, 2, d), (far, d, 1))
    kv[:, 0], kv[:, 1] = k[:, 0].cuda(), v[:, 0].cuda()
    n = [rows - 65, 65]
    want, tol = reference(q, split(k, n), split(v, n), n, n, 0.125, True)
    for most in (rows, 400):     # one group of wavefronts, two
        out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
        desc = packed_desc(2, 2, 1, d, rows, rows, most, most, True, 0.125, None, [far, 0], [far, 0])
        attend_packed(device, desc, q.cuda(), kv, kv[:, 1:], starts_of(n).cuda(), None, out)
        close(out, want, tol, most)


@gpu
@pytest.mark.parametrize("heads,kv_heads,d,causal,n", [(32, 8, 128, True, [700, 300, 1000]), (6, 6, 64, False, [600, 500]), (4, 1, 96, True, [1500]), (40, 40, 40, True, [300, 10]), (2, 2, 128, False, [900])])
def test_longer_prompts(device, heads, kv_heads, d, causal, n):
    """One and two groups of wavefronts, one and several shares."""
    run(device, heads, n, heads, kv_heads, d, causal)


@gpu
def test_without_starts_every_sequence_has_as_many_rows(device):
    b, n, heads, d = 3, 77, 2, 64
    q, k, v = inputs(11, b * n, b * n, heads, heads, d)
    want, tol = reference(q, split(k, [n] * b), split(v, [n] * b), [n] * b, [n] * b, 0.125, True)
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    attend_packed(device, packed_desc(b, heads, heads, d, b * n, b * n, n, n, True, 0.125), q.cuda(), k.cuda(), v.cuda(), None, None, out)
    close(out, want, tol)
    again = torch.empty_like(out)   # and with keys of their own
    attend_packed(device, packed_desc(b, heads, heads, d, b * n, b * n, n, n, True, 0.125), q.cuda(), k.cuda(), v.cuda(), None, starts_of([n] * b).cuda(), again)
    assert torch.equal(out, again)


@gpu
def test_rows_past_the_bounds_are_left(device):
    """starts that promise more than max_rows, point outside the tensor, or descend: nothing outside is read or written."""
    q, k, v = (x.cuda() for x in inputs(12, 100, 100, 1, 1, 64))
    for starts, left in (([0, 100], 60), ([-5, 30, 400], 100), ([40, 10, 90], 100)):
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
        attend_packed(device, packed_desc(len(starts) - 1, 1, 1, 64, 100, 100, 60, 100, True, 0.125), q, k, v, torch.tensor(starts, dtype=torch.int32, device="cuda"), None, out)
        assert bool((out[left:] == 7.0).all()) and bool(torch.isfinite(out[10:30]).all())


@gpu
def test_the_same_call_gives_the_same_bits_and_graphs_take_new_lengths(device):
    heads, kv, d, rows = 4, 2, 128, 400
    q, k, v = (x.cuda() for x in inputs(13, rows, rows, heads, kv, d))
    starts = starts_of([100, 300]).cuda()
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    desc = packed_desc(2, heads, kv, d, rows, rows, rows, rows, True, 0.09)
    need = ctypes.c_uint64()
    assert _ffi.lib().rt_attention_packed_workspace_bytes(desc, need) == _ffi.RT_OK
    ws = torch.zeros(max(need.value, 1), dtype=torch.uint8, device="cuda")
    attend_packed(device, desc, q, k, v, starts, None, out, ws)
    first = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        attend_packed(device, desc, q, k, v, starts, None, out, ws)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        attend_packed(device, desc, q, k, v, starts, None, out, ws)
    for sizes in ([100, 300], [1, 399], [250, 0], [400, 0], [100, 300]):
        starts.copy_(starts_of(sizes))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(out, 7.0)
        attend_packed(device, desc, q, k, v, starts, None, eager, ws)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        if sizes == [100, 300]:
            assert torch.equal(out, first)


# ---- what is refused: no GPU is needed ---------------------------------------------------------------------------------------


def fine():
    return packed_desc(2, 8, 2, 64, 10, 10, 8, 8, True, 0.125)


@pytest.mark.parametrize("field,value,status", [
    ("batch", -1, _ffi.RT_ERR_INVALID_SHAPE), ("heads", -8, _ffi.RT_ERR_INVALID_SHAPE), ("kv_heads", 3, _ffi.RT_ERR_INVALID_SHAPE), ("kv_heads", 0, _ffi.RT_ERR_INVALID_SHAPE),
    ("kv_heads", -2, _ffi.RT_ERR_INVALID_SHAPE), ("head_dim", 0, _ffi.RT_ERR_INVALID_SHAPE), ("head_dim", 60, _ffi.RT_ERR_INVALID_SHAPE), ("head_dim", 136, _ffi.RT_ERR_INVALID_SHAPE),
    ("rows", -1, _ffi.RT_ERR_INVALID_SHAPE), ("kv_rows", -1, _ffi.RT_ERR_INVALID_SHAPE), ("max_rows", -1, _ffi.RT_ERR_INVALID_SHAPE), ("max_keys", -1, _ffi.RT_ERR_INVALID_SHAPE),
    ("causal", 2, _ffi.RT_ERR_INVALID_ARG), ("scale", float("nan"), _ffi.RT_ERR_INVALID_ARG), ("scale", float("inf"), _ffi.RT_ERR_INVALID_ARG),
    ("rows", (1 << 25) + 1, _ffi.RT_ERR_UNSUPPORTED), ("max_keys", (1 << 30) + 1, _ffi.RT_ERR_UNSUPPORTED), ("batch", 65536, _ffi.RT_ERR_UNSUPPORTED),
    ("heads", 1 << 29, _ffi.RT_ERR_UNSUPPORTED), ("heads", (1 << 20) + 2, _ffi.RT_ERR_UNSUPPORTED),
])
def test_refusals(field, value, status):
    L, d, need = _ffi.lib(), fine(), ctypes.c_uint64()
    assert L.rt_attention_packed_validate(d) == _ffi.RT_OK
    setattr(d, field, value)
    assert L.rt_attention_packed_validate(d) == status
    assert L.rt_attention_packed_workspace_bytes(d, need) == status


def test_rows_times_heads():
    """Tiles of 128 rows past the last one still have numbers of 31 bits."""
    for rows, status in (((1 << 25) - 1, _ffi.RT_ERR_UNSUPPORTED), ((1 << 25) - 4, _ffi.RT_OK)):
        d = packed_desc(1, 64, 64, 8, rows, rows, 1, 1, True, 0.1)
        d.max_rows = 128
        assert _ffi.lib().rt_attention_packed_validate(d) == status, rows


@pytest.mark.parametrize("name", ["q_strides", "k_strides", "v_strides", "o_strides"])
def test_refused_strides(name):
    for i in range(2):
        for value, status in ((-8, _ffi.RT_ERR_INVALID_SHAPE), (12, _ffi.RT_OK if name == "o_strides" else _ffi.RT_ERR_UNSUPPORTED), (1 << 40, _ffi.RT_ERR_UNSUPPORTED)):
            d = fine()
            getattr(d, name)[i] = value
            assert _ffi.lib().rt_attention_packed_validate(d) == status, (i, value)


def test_null_arguments():
    L, need = _ffi.lib(), ctypes.c_uint64()
    assert L.rt_attention_packed_validate(None) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_packed_workspace_bytes(None, need) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_packed_workspace_bytes(fine(), None) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_packed_enqueue(None, fine(), None, None, None, None, None, None, None, 0, None) == _ffi.RT_ERR_INVALID_ARG


@gpu
def test_refused_calls(device):
    L = _ffi.lib()
    z = torch.zeros(10 * 8 * 64 + 8, dtype=torch.float16, device="cuda")
    s = torch.zeros(8, dtype=torch.int32, device="cuda")
    good = [device.ctx, fine(), z.data_ptr(), z.data_ptr(), z.data_ptr(), s.data_ptr(), None, z.data_ptr(), None, 0, None]
    for at, value, status in ((2, None, 1), (3, None, 1), (4, None, 1), (7, None, 1), (2, z.data_ptr() + 2, 1), (3, z.data_ptr() + 8, 1), (4, z.data_ptr() + 8, 1),
                              (5, s.data_ptr() + 2, 1), (6, s.data_ptr() + 1, 1), (7, z.data_ptr() + 1, 1), (5, None, 2)):
        args = list(good)
        args[at] = value
        assert L.rt_attention_packed_enqueue(*args) == status, at
    d = fine()
    d.kv_rows = 9      # without kv_starts the keys are where the queries are
    assert L.rt_attention_packed_enqueue(*(good[:1] + [d] + good[2:])) == _ffi.RT_ERR_INVALID_SHAPE
    for field in ("batch", "rows", "max_rows"):
        d = packed_desc(0 if field == "batch" else 2, 8, 2, 64, 0 if field == "rows" else 10, 0 if field == "rows" else 10, 0 if field == "max_rows" else 8, 8, True, 0.1)
        assert L.rt_attention_packed_enqueue(device.ctx, d, None, None, None, s.data_ptr(), None, None, None, 0, None) == _ffi.RT_OK   # nothing to do
    torch.cuda.synchronize()
    assert not bool(z.any())
