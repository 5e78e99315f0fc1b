"""Attention over 4-bit caches where its kernels meet their limits: shares of a long axis and how they are joined, moving maxima, small probabilities, tiles that end
inside a share, outputs that start anywhere, graphs, streams, caches past 4 GiB.  Reference and tolerance are those of test_cache_q4."""
import ctypes

import numpy as np
import pytest
import torch

from ratchet_amd import _ffi
from test_cache_q4 import DIMS, attention_desc, blocks, buffer, check, drawn_cache, held, reference, run, values

gpu = pytest.mark.gpu
ROWS = [1, 3, 6, 13, 17, 40, 150]  # query rows of one head: each number of result registers, one wavefront's rows, several, several tiles


def workspace_bytes(*a, **k):
    need = ctypes.c_uint64()
    assert _ffi.lib().rt_attention_q4_workspace_bytes(ctypes.byref(attention_desc(*a, **k)), ctypes.byref(need)) == 0
    return need.value


def test_workspace_follows_the_shape():
    """One launch for short caches and where the rows fill the device; shares elsewhere, of at most 256 per row; no size below zero or past its rows."""
    assert workspace_bytes(1, 32, 32, 1, 1024, 80, 1024) == 0
    assert workspace_bytes(32, 32, 8, 1, 8192, 128, 8192) == 0
    assert workspace_bytes(1, 32, 32, 2048, 2048, 96, 2048) == 0
    for b, h, kv, lq, n, d in ((1, 32, 8, 1, 32768, 128), (1, 8, 1, 1, 1 << 20, 128), (2, 16, 4, 150, 1373, 64), (1, 8, 2, 64, 8192, 64), (1, 1, 1, 17, 1 << 30, 16)):
        need, row = workspace_bytes(b, h, kv, lq, n, d, n), b * h * lq * (d + 2) * 4
        assert need % row == 0 and 2 <= need // row <= 256, (need, row)
    for n in (0, 1, 512, 513):
        assert workspace_bytes(1, 4, 4, 1, n, 64, n) == 0


@gpu
@pytest.mark.parametrize("lq", ROWS)
@pytest.mark.parametrize("top", [4.0, 5.2, 10.7])
def test_one_large_probability_and_many_small_ones(device, lq, top):
    """exp(-10.7) = 2^-15.4 is a subnormal f16, 6000 of which weigh an eighth of the one; 5.2 leaves them below 2^-7.5, where a reference of theirs need not move for the one.
    The large score comes first, last, or at the end of the first block."""
    rng = np.random.default_rng(lq)
    n, d = 6000, 64
    for at in (0, n - 1, 63):
        codes, ds = np.full((1, 1, n, d), 8, np.uint8), np.full((1, 1, n, 2), 0.5, np.float16)
        codes[0, 0, at, 0] = 12  # 2 in dimension 0
        vcodes, vds = rng.integers(0, 16, (1, 1, n, d), dtype=np.uint8), np.full((1, 1, n, 2), 0.25, np.float16)
        q = np.zeros((1, 1, lq, d), np.float16)
        q[..., 0] = np.linspace(1, 1.01, lq)
        scale = np.float32(top / 2)
        want, tol = reference(q, values(codes, ds), values(vcodes, vds), float(scale))
        for ws in (True, False):
            check(run(device, q, buffer(codes, ds), buffer(vcodes, vds), 1, n, n, scale, workspace=ws), want, tol)


@gpu
@pytest.mark.parametrize("lq", ROWS)
@pytest.mark.parametrize("slope", [0.02, -0.02, 0.4])
def test_scores_that_rise_and_fall_along_the_keys(device, lq, slope):
    """The maximum moves in every block, or never again; differences past what an exponential holds."""
    rng = np.random.default_rng(3)
    n, d = 1500, 96
    codes, ds = rng.integers(0, 16, (1, 2, n, d), dtype=np.uint8), np.full((1, 2, n, 3), 2.0**-6, np.float16)
    codes[..., :32] = 8
    codes[..., 0] = 9
    ds[..., 0] = (np.arange(n) - n / 2 if slope > 0 else n / 2 - np.arange(n)).astype(np.float16)  # dimension 0 is the key's number
    vbuf, vval = drawn_cache(rng, 1, 2, n, d)
    q = rng.standard_normal((1, 2, lq, d)).astype(np.float16)
    q[..., 0] = abs(slope)
    want, tol = reference(q, values(codes, ds), vval, 1.0)
    wc, tc = reference(q, values(codes, ds), vval, 1.0, causal=True)
    for ws in (True, False):
        check(run(device, q, buffer(codes, ds), vbuf, 2, n, n, 1.0, workspace=ws), want, tol)
        check(run(device, q, buffer(codes, ds), vbuf, 2, n, n, 1.0, causal=True, workspace=ws), wc, tc)


# (batch, heads, kv_heads, query rows, keys): shares that end inside a block, one key past a share, tiles whose last rows see a share and whose first do not
LONG = [(1, 2, 1, 1, 5000), (1, 4, 1, 1, 1025), (1, 8, 1, 1, 1537), (1, 3, 1, 5, 2049), (1, 2, 2, 20, 1300), (1, 2, 1, 64, 1281), (2, 4, 2, 150, 1373), (1, 1, 1, 300, 897)]


@gpu
@pytest.mark.parametrize("d", DIMS)
def test_shares_of_a_long_axis(device, d):
    rng = np.random.default_rng(d)
    for b, h, kv, lq, n in LONG if d in (64, 128) else LONG[1::2]:
        cap = n + 3
        kbuf, kval = drawn_cache(rng, b, kv, cap, d, garbage_from=n)
        vbuf, vval = drawn_cache(rng, b, kv, cap, d, garbage_from=n)
        q = rng.standard_normal((b, h, lq, d)).astype(np.float16)
        lens = [n - 400 * i for i in range(b)]
        assert workspace_bytes(b, h, kv, lq, n, d, cap) > 0
        for causal, ls in ((False, None), (True, None), (True, lens), (True, [lq // 2] * b)):
            want, tol = reference(q, kval[:, :, :n], vval[:, :, :n], 0.2, causal=causal, lens=ls)
            for ws in (True, False):
                check(run(device, q, kbuf, vbuf, kv, cap, n, 0.2, causal=causal, lens=ls, workspace=ws), want, tol)


@gpu
@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("d", [48, 80, 112, 128])
@pytest.mark.parametrize("lq", [4, 8, 16, 45])
def test_masks_of_odd_rows_over_long_caches(device, dt, d, lq):
    """Rows of masks that start on no vector, over several shares; a query that is not finite spoils its row and, through hidden keys, no other."""
    rng = np.random.default_rng(d + lq)
    h, n = 2, 1301
    kbuf, kval = drawn_cache(rng, 1, h, n, d)
    vbuf, vval = drawn_cache(rng, 1, h, n, d)
    q = rng.standard_normal((1, h, lq, d)).astype(np.float16)
    mask = np.where(rng.random((lq, n)) < 0.3, -np.inf, rng.uniform(-4, 4, (lq, n))).astype(dt)
    mask[0, : n - 1] = np.finfo(dt).min
    mask[1, 1:] = -np.inf
    mask[2] = -np.inf
    want, tol = reference(q, kval, vval, 0.2, mask=mask)
    for ws in (True, False):
        got = run(device, q, kbuf, vbuf, h, n, n, 0.2, mask=mask, workspace=ws)
        check(got, want, tol)
    q[0, 1, 3, 5] = np.inf
    got = run(device, q, kbuf, vbuf, h, n, n, 0.2, mask=mask)
    assert np.isnan(got[0, 1, 3]).all()
    want[0, 1, 3] = np.nan
    check(got, want, tol)


@gpu
@pytest.mark.parametrize("lq", [1, 6, 20, 130])
def test_keys_that_are_not_finite_behind_a_mask(device, lq):
    """Hidden by a mask tensor in one tile of a long cache, seen in another."""
    rng = np.random.default_rng(lq)
    n, d = 1100, 112
    codes, ds = rng.integers(0, 16, (1, 2, n, d), dtype=np.uint8), np.full((1, 2, n, blocks(d)), 0.125, np.float16)
    kds, vds = ds.copy(), ds.copy()
    bad = [5, 127, 128, 700, 1099]
    kds[0, :, bad, 1], vds[0, :, bad, 3] = np.nan, np.inf
    mask = rng.uniform(-2, 2, (lq, n)).astype(np.float32)
    mask[:, bad] = -np.inf
    q = rng.standard_normal((1, 2, lq, d)).astype(np.float16)
    zero = lambda x: values(codes, np.where(np.isfinite(x), x, 0))
    want, tol = reference(q, zero(kds), zero(vds), 0.1, mask=mask)
    for ws in (True, False):
        check(run(device, q, buffer(codes, kds), buffer(codes, vds), 2, n, n, 0.1, mask=mask, workspace=ws), want, tol)
    mask[lq - 1, 700] = 0  # the last row sees one of them
    got = run(device, q, buffer(codes, kds), buffer(codes, vds), 2, n, n, 0.1, mask=mask)
    assert np.isnan(got[0, :, lq - 1]).all()
    check(got[:, :, : lq - 1], want[:, :, : lq - 1], tol[:, :, : lq - 1])


@gpu
@pytest.mark.parametrize("lq", [1, 9, 21])
def test_outputs_and_queries_anywhere(device, lq):
    """Outputs that start on odd elements with rows an odd number apart; queries a head's row apart from one another; nothing else is written."""
    rng = np.random.default_rng(lq)
    b, h, kv, n, d = 2, 4, 2, 700, 80
    kbuf, kval = drawn_cache(rng, b, kv, n, d)
    vbuf, vval = drawn_cache(rng, b, kv, n, d)
    q = rng.standard_normal((b, h, lq, d)).astype(np.float16)
    want, tol = reference(q, kval, vval, 0.2)
    desc = attention_desc(b, h, kv, lq, n, d, n, 0, 0.2)
    qs, os = [h * (d + 16) * lq, (d + 16) * lq, d + 16], [lq * (d + 3) * h + 5, lq * (d + 3), d + 3]
    desc.q_strides[:], desc.o_strides[:] = qs, os
    qt = torch.full((b * qs[0],), float("nan"), dtype=torch.float16, device="cuda:0")
    qt.as_strided((b, h, lq, d), (*qs, 1)).copy_(torch.from_numpy(q))
    out = torch.full((b * os[0] + 1,), 7.0, dtype=torch.float16, device="cuda:0")
    to = lambda x: torch.from_numpy(x).to("cuda:0")
    k, v = to(kbuf), to(vbuf)
    st = _ffi.lib().rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), qt.data_ptr(), k.data_ptr(), v.data_ptr(), None, None, out.data_ptr() + 2, None, 0,
                                            torch.cuda.current_stream().cuda_stream)
    assert st == 0
    got = out[1:].as_strided((b, h, lq, d), (*os, 1))
    check(got.cpu().numpy(), want, tol)
    got.fill_(7)
    assert (out == 7).all()


@gpu
@pytest.mark.parametrize("lq", [1, 40])
def test_steps_captured_into_a_graph(device, lq):
    """A write at offsets and an attention over lengths from the device, captured once on another stream and replayed as they grow: every replay is the eager result, bit for bit."""
    rng = np.random.default_rng(8)
    b, h, kv, cap, d = 2, 8, 2, 4000, 64
    L, need = _ffi.lib(), ctypes.c_uint64()
    desc = attention_desc(b, h, kv, lq, cap, d, cap, 1)
    assert L.rt_attention_q4_workspace_bytes(ctypes.byref(desc), ctypes.byref(need)) == 0 and need.value > 0
    gpu_ = lambda x: torch.from_numpy(x).to("cuda:0")
    caches = [gpu_(drawn_cache(rng, b, kv, cap, d)[0]) for _ in range(2)]
    q, k, v = (gpu_(rng.standard_normal((b, n, lq, d)).astype(np.float16)) for n in (h, kv, kv))
    desc.q_strides[:] = desc.o_strides[:] = [h * lq * d, lq * d, d]
    at = torch.zeros(b, dtype=torch.int32, device="cuda:0")

    def step(caches, at, ws, out, stream):
        strides = (ctypes.c_int64 * 3)(kv * lq * d, lq * d, d)
        lens = at + lq
        assert L.rt_cache_write_q4_enqueue(device.ctx, _ffi.RT_F16, caches[0].data_ptr(), k.data_ptr(), caches[1].data_ptr(), v.data_ptr(), strides, None, None,
                                           at.data_ptr(), b, kv, cap, 0, lq, d, stream) == 0
        assert L.rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), q.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), None, lens.data_ptr(),
                                         out.data_ptr(), ws.data_ptr(), need.value, stream) == 0

    mine, eager = [[c.clone() for c in caches] for _ in range(2)]
    ws = [torch.empty(need.value, dtype=torch.uint8, device="cuda:0") for _ in range(2)]
    out = [torch.empty((b, h, lq, d), dtype=torch.float16, device="cuda:0") for _ in range(2)]
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(mine, at, ws[0], out[0], torch.cuda.current_stream().cuda_stream)
    for lens in ([0, 0], [3, 700], [1500, 64], [cap - lq, 2047], [cap - 1, cap]):
        at.copy_(torch.tensor(lens, dtype=torch.int32))
        q.mul_(0.9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(eager, at, ws[1], out[1], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(mine, eager)), lens
        assert torch.equal(out[0].view(torch.int16), out[1].view(torch.int16)) and torch.isfinite(out[0]).all(), lens


@gpu
def test_a_cache_past_four_gigabytes(device):
    """The second head's rows, and their scales, start beyond 2^32 bytes of the buffer; written there and read there."""
    rng = np.random.default_rng(5)
    h, cap, d, n = 2, (1 << 26) + 1000, 128, 700
    L = _ffi.lib()
    nbytes, soff = ctypes.c_uint64(), ctypes.c_uint64()
    assert L.rt_cache_q4_nbytes(1, h, cap, d, ctypes.byref(nbytes), ctypes.byref(soff)) == 0 and cap * d // 2 > 1 << 32
    cache = torch.zeros(nbytes.value, dtype=torch.uint8, device="cuda:0")
    rows = rng.standard_normal((1, h, n, d)).astype(np.float16)
    src = torch.from_numpy(rows).to("cuda:0")
    stream = torch.cuda.current_stream().cuda_stream
    strides = (ctypes.c_int64 * 3)(h * n * d, n * d, d)
    write = lambda offset: L.rt_cache_write_q4_enqueue(device.ctx, _ffi.RT_F16, cache.data_ptr(), src.data_ptr(), None, None, strides, None, None, None, 1, h, cap, offset,
                                                       n, d, stream)
    assert write(0) == 0 and write(cap - n) == 0
    val = held(rows)[2]
    codes = lambda head, row: cache[(head * cap + row) * d // 2 :][: n * d // 2]
    sc = lambda head, row: cache[soff.value + (head * cap + row) * 8 :][: n * 8]
    for head in range(h):  # the same rows at both ends of a head, and nothing behind them
        assert torch.equal(codes(head, 0), codes(head, cap - n)) and torch.equal(sc(head, 0), sc(head, cap - n)) and bool(codes(head, 0).any())
        assert not bool(codes(head, n).any()) and not bool(sc(head, n).any())
    for lq in (1, 20):
        q = rng.standard_normal((1, h, lq, d)).astype(np.float16)
        want, tol = reference(q, val, val, 0.1)
        desc = attention_desc(1, h, h, lq, n, d, cap, 0, 0.1, heads_inside=False)
        qt, out = torch.from_numpy(q).to("cuda:0"), torch.zeros((1, h, lq, d), dtype=torch.float16, device="cuda:0")
        assert L.rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), qt.data_ptr(), cache.data_ptr(), cache.data_ptr(), None, None, out.data_ptr(), None, 0, stream) == 0
        check(out.cpu().numpy(), want, tol)
    # all rows of the heads, most of them zeros: keys 0 and values 0, and the written ones far behind a 32-bit offset from the head's first
    q = np.zeros((1, h, 1, d), np.float16)
    q[..., 0] = 8
    desc = attention_desc(1, h, h, 1, cap, d, cap, 0, 1.0, heads_inside=False)
    need = ctypes.c_uint64()
    assert L.rt_attention_q4_workspace_bytes(ctypes.byref(desc), ctypes.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda:0")
    qt, out = torch.from_numpy(q).to("cuda:0"), torch.zeros((1, h, 1, d), dtype=torch.float16, device="cuda:0")
    assert L.rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), qt.data_ptr(), cache.data_ptr(), cache.data_ptr(), None, None, out.data_ptr(), ws.data_ptr(), need.value,
                                     stream) == 0
    # zeros beside them: exp(0) each, which the two copies' sums have to be weighed against
    s = val[0, :, :, 0] * 8
    p = np.exp(s)
    want = 2 * (p[..., None] * val[0]).sum(1) / (2 * p.sum(1) + cap - 2 * n)[:, None]
    mag = 2 * (p[..., None] * np.abs(val[0])).sum(1) / (2 * p.sum(1) + cap - 2 * n)[:, None]
    # the sum's f32 terms: at most 2^11 steps of a lane, half of 2^-24 each on average; a score's error as elsewhere; the f16 probabilities' below their normal range
    e = (d / 32 + 36) * 2.0**-23 * np.abs(s).max()
    assert (np.abs(out[0, :, 0].double().cpu().numpy() - want) <= (2.0**-11 + 2.0**-14 + 2.0**-20 + 4 * e) * mag + 2.0**-11 * np.abs(want) + 2.0**-25
            + 2.0**-25 * 2 * np.abs(val[0]).sum(1)).all()


@gpu
@pytest.mark.parametrize("lq", [1, 2])
def test_one_workgroup_past_its_window(device, lq):
    """Without a workspace one workgroup has all the keys, more than the 2^24 that its offsets are counted in: two keys, one on each side of that line and each with values of
    its own, have the same largest score."""
    rng = np.random.default_rng(6)
    n, d = (1 << 24) + 700, 16
    some = np.concatenate([np.arange(40), (1 << 24) + np.arange(-30, 40), n - 1 - np.arange(20)])
    q = rng.standard_normal((1, 1, lq, d)).astype(np.float16)
    q[0, 0] = q[0, 0, 0]
    kc, vc = np.full((n, d), 8, np.uint8), np.full((n, d), 8, np.uint8)
    kd, vd = np.zeros((n, 1), np.float16), np.zeros((n, 1), np.float16)
    kc[some], kd[some, 0] = rng.integers(0, 16, (len(some), d)), rng.uniform(0.1, 0.2, len(some))
    vc[some], vd[some, 0] = rng.integers(0, 16, (len(some), d)), rng.uniform(0.2, 0.5, len(some))
    for at in (5, (1 << 24) + 11):
        kc[at], kd[at, 0] = np.where(q[0, 0, 0] > 0, 12, 4), 0.5
    kv, vv = values(kc[some], kd[some]), values(vc[some], vd[some])
    got = run(device, q, buffer(kc[None, None], kd[None, None]), buffer(vc[None, None], vd[None, None]), 1, n, n, 1.0, workspace=False)[0, 0].astype(np.float64)
    x = q[0, 0, 0].astype(np.float64)
    s = kv @ x
    p = np.exp(s - s.max())
    zeros = (n - len(some)) * np.exp(-s.max())
    l = p.sum() + zeros
    assert (p > 0.99).sum() == 2 and zeros < 0.5
    e = (d / 32 + 36) * 2.0**-23 * (np.abs(kv) @ np.abs(x)).max() + 2.0**-22 * s.max()
    want, mag = p @ vv / l, p @ np.abs(vv) / l
    # beside what holds elsewhere: the sum, in f32 over 2^15 steps of a lane, off by at most half a step of a partial sum that grows evenly: 2^-10 of the zeros' part
    tol = (2.0**-11 + 2.0**-20 + 2 * e) * mag + 2.0**-25 * np.abs(vv).sum(0) / l + 2.0**-11 * np.abs(want) + 2.0**-25 + 2.0**-10 * zeros / l * np.abs(want)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@gpu
@pytest.mark.parametrize("lq", [1, 20])
def test_no_keys_and_no_caches(device, lq):
    """kv_len = 0: every row is NaN, and the caches may be NULL."""
    desc = attention_desc(2, 4, 2, lq, 0, 64, 8)
    q = torch.zeros((2, lq, 4, 64), dtype=torch.float16, device="cuda:0")
    out = torch.zeros_like(q)
    for causal in (0, 1):
        desc.causal = causal
        out.zero_()
        assert _ffi.lib().rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), q.data_ptr(), None, None, None, None, out.data_ptr(), None, 0,
                                                  torch.cuda.current_stream().cuda_stream) == 0
        assert torch.isnan(out).all()


@gpu
@pytest.mark.parametrize("lq", [1, 5, 17])
def test_as_many_sequences_as_a_call_takes(device, lq):
    """65535 heads of keys in one call; one more is refused."""
    rng = np.random.default_rng(lq)
    b, kv, n, d = 13107, 5, 3, 16
    kbuf, kval = drawn_cache(rng, b, kv, n, d)
    vbuf, vval = drawn_cache(rng, b, kv, n, d)
    q = rng.standard_normal((b, kv, lq, d)).astype(np.float16)
    got = run(device, q, kbuf, vbuf, kv, n, n, 0.2)
    for i in (0, 1, 6000, b - 1):
        want, tol = reference(q[i : i + 1], kval[i : i + 1], vval[i : i + 1], 0.2)
        check(got[i : i + 1], want, tol)
    desc = attention_desc(65536, 1, 1, lq, n, d, n)
    assert _ffi.lib().rt_attention_q4_validate(ctypes.byref(desc)) == _ffi.RT_ERR_UNSUPPORTED


@gpu
@pytest.mark.parametrize("h,kv,lq", [(64, 1, 1), (16, 1, 1), (17, 1, 1), (40, 8, 3), (64, 2, 9)])
def test_many_heads_on_one(device, h, kv, lq):
    """Groups that make a tile of one query row, that fill the streaming kernel's rows and that pass them by one; a mask's row belongs to all heads of its query."""
    rng = np.random.default_rng(h)
    b, n, d = 2, 640, 80
    kbuf, kval = drawn_cache(rng, b, kv, n, d)
    vbuf, vval = drawn_cache(rng, b, kv, n, d)
    q = rng.standard_normal((b, h, lq, d)).astype(np.float16)
    mask = np.where(rng.random((b, lq, n)) < 0.3, -np.inf, rng.uniform(-2, 2, (b, lq, n))).astype(np.float16)
    for causal, m, lens in ((False, None, None), (True, None, [600, 11]), (True, mask, None)):
        want, tol = reference(q, kval, vval, 0.2, mask=m, causal=causal, lens=lens)
        check(run(device, q, kbuf, vbuf, kv, n, n, 0.2, mask=m, causal=causal, lens=lens), want, tol)


@gpu
@pytest.mark.parametrize("h,lq,n,d", [(4, 1, 70000, 128), (1, 6, 33281, 48), (16, 1, 131072, 64), (1, 1, 66000, 16)])
def test_more_shares_than_a_join_reads_at_once(device, h, lq, n, d):
    """One head of keys on the whole device: 66 to 256 shares of a row, joined 64 at a time; the largest scores in the last."""
    rng = np.random.default_rng(n)
    kbuf, kval = drawn_cache(rng, 1, 1, n, d)
    vbuf, vval = drawn_cache(rng, 1, 1, n, d)
    q = rng.standard_normal((1, h, lq, d)).astype(np.float16)
    assert workspace_bytes(1, h, 1, lq, n, d, n) // (h * lq * (d + 2) * 4) > 64
    mask = np.zeros((lq, n), np.float32)
    mask[:, -300:] = 12
    for m, lens in ((None, None), (mask, None), (None, [n - 20000])):
        want, tol = reference(q, kval, vval, 0.1, mask=m, lens=lens)
        check(run(device, q, kbuf, vbuf, 1, n, n, 0.1, mask=m, lens=lens), want, tol)
