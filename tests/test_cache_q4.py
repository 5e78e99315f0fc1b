"""The key/value cache held in 4-bit blocks and the attention over it, against numpy in float64.

The format is restated here from its definition (held): bytes and values of the write have to be equal.  The caches of the attention tests are drawn as
codes and scales, or written by the library's own write.

Tolerance of the attention.  Scores: codes, scales and queries are exact in f32, so a score s of D products and D / 32 scaled sums is off by at most
(D / 32 + 36) 2^-23 sum_c |scale q k| (2^-23 each for the matrix cores' own order and truncation), and with the mask's addition and the step to base 2 by 4 * 2^-24 of
|s| + |mask| more; that shifts a probability by as much relatively, e in all below.  A probability is rounded to f16 (2^-11 relative, 2^-25 below 2^-14;
it is at most 1 against the largest), the hardware exponential is within 2^-21; the output is a mean of values with these weights, so it is off by at most
(2^-11 + 2 e + 2^-20) sum_j w |v| + 2^-25 sum_j |v| / l, l >= 1 the sum of the probabilities against their maximum, and by the rounding to f16: 2^-11 |out| + 2^-25."""
import ctypes

import numpy as np
import pytest
import torch

from ratchet_amd import DType, Device, InvariantError, OperationError, Tensor, _ffi, nn
from ratchet_amd.tensor import cache_q4_nbytes

gpu = pytest.mark.gpu
DIMS = [16, 32, 48, 64, 80, 96, 112, 128]


def blocks(d):
    return (d + 31) // 32


def scales(d):
    return {1: 1, 2: 2, 3: 4, 4: 4}[blocks(d)]


def held(x):
    """f16 rows [..., D] -> codes [..., D], f16 scales [..., blocks], values [..., D] in float64."""
    d = x.shape[-1]
    codes, ds = np.zeros(x.shape, np.uint8), np.zeros(x.shape[:-1] + (blocks(d),), np.float16)
    x = x.astype(np.float64)
    for k in range(blocks(d)):
        z = x[..., 32 * k : min(d, 32 * k + 32)]
        m = np.take_along_axis(z, np.abs(z).argmax(-1)[..., None], -1)[..., 0]  # argmax: the first of equals
        t = np.abs(m) / 8
        unit = np.ldexp(1.0, np.maximum(np.frexp(t)[1] - 8, -24))
        s = np.minimum(np.round(t / unit) * unit, 8160.0) * -np.sign(m)  # np.round: ties to even
        with np.errstate(invalid="ignore", divide="ignore"):
            q = np.where(s[..., None] == 0, 8, np.clip(np.floor(z / s[..., None] + 8.5), 0, 15))
        bad = ~np.isfinite(z).all(-1)
        q[bad], s[bad] = 8, np.nan
        codes[..., 32 * k : 32 * k + z.shape[-1]], ds[..., k] = q, s
    return codes, ds, values(codes, ds)


def values(codes, ds):
    return (codes.astype(np.float64) - 8) * np.repeat(ds.astype(np.float64), 32, -1)[..., : codes.shape[-1]]


def packed(codes):
    out = np.zeros(codes.shape[:-1] + (codes.shape[-1] // 8,), np.uint32)
    for e in range(8):
        out |= codes[..., e::8].astype(np.uint32) << np.uint32(4 * (e // 2 + 4 * (e % 2)))
    return out.view(np.uint8)


def buffer(codes, ds):
    """The bytes of a cache: codes [b, h, capacity, D], scales [b, h, capacity, blocks]."""
    d = codes.shape[-1]
    wide = np.zeros(ds.shape[:-1] + (scales(d),), np.float16)
    wide[..., : blocks(d)] = ds
    pad = lambda b: np.concatenate([b, np.zeros(-len(b) % 256, np.uint8)])
    return np.concatenate([pad(packed(codes).reshape(-1)), pad(wide.view(np.uint8).reshape(-1))])


def cache_tensor(buf, shape, device):
    t = Tensor(shape, DType.Q4_0, device, torch.from_numpy(buf).to(device.torch_device()))
    t.is_q4_cache = True
    return t


# ---- on the CPU -----------------------------------------------------------------------------------------------------------


def test_sizes():
    n, at = ctypes.c_uint64(), ctypes.c_uint64()
    for d in DIMS:
        for shape in [(1, 1, 1), (2, 3, 17), (0, 4, 8), (1, 2, 0), (3, 5, 1000)]:
            assert cache_q4_nbytes((*shape, d)) == (len(buffer(np.zeros((*shape, d), np.uint8), np.zeros((*shape, blocks(d)), np.float16))),
                                                    (int(np.prod(shape)) * d // 2 + 255) // 256 * 256)
    f = _ffi.lib().rt_cache_q4_nbytes
    for bad in [(1, 1, 1, 0), (1, 1, 1, 8), (1, 1, 1, 72), (1, 1, 1, 144), (-1, 1, 1, 64), (1, 1, -1, 64)]:
        assert f(*bad, ctypes.byref(n), ctypes.byref(at)) == _ffi.RT_ERR_INVALID_SHAPE
    assert f(1, 1, 1, 64, None, None) == _ffi.RT_ERR_INVALID_ARG
    assert f(65535, 1, 0x7fffffff, 128, ctypes.byref(n), ctypes.byref(at)) == 0 and n.value > 2**52  # (no wrap)


def attention_desc(b, h, kv, lq, kv_len, d, cap, causal=0, scale=None, mask=None, heads_inside=True):
    x = _ffi.AttentionQ4Desc()
    x.batch, x.heads, x.kv_heads, x.q_len, x.kv_len, x.head_dim, x.capacity, x.causal = b, h, kv, lq, kv_len, d, cap, causal
    x.q_strides[:] = [lq * h * d, d, h * d] if heads_inside else [h * lq * d, lq * d, d]
    x.o_strides[:] = x.q_strides[:]
    x.scale = 1 / np.sqrt(max(d, 1)) if scale is None else scale
    if mask is not None:
        x.mask_dtype = _ffi.RT_F16 if mask.dtype == np.float16 else _ffi.RT_F32
        x.mask_strides[:] = [mask.shape[-1] * lq if mask.ndim == 3 else 0, mask.shape[-1]]
    return x


def test_attention_descriptor_rules():
    L, need = _ffi.lib(), ctypes.c_uint64()
    ok = lambda **k: L.rt_attention_q4_validate(ctypes.byref(changed(**k)))

    def changed(**k):
        d = attention_desc(2, 8, 4, 3, 50, 64, 60)
        for name, v in k.items():
            if isinstance(v, tuple):
                getattr(d, name)[v[0]] = v[1]
            else:
                setattr(d, name, v)
        return d

    assert ok() == 0 and L.rt_attention_q4_validate(None) == _ffi.RT_ERR_INVALID_ARG
    for k in (dict(kv_heads=3), dict(kv_heads=0), dict(head_dim=72), dict(head_dim=144), dict(head_dim=0), dict(kv_len=61), dict(kv_len=-1), dict(q_len=-1),
              dict(batch=-1), dict(q_strides=(0, -8)), dict(o_strides=(2, -1)), dict(mask_strides=(1, -1))):
        assert ok(**k) == _ffi.RT_ERR_INVALID_SHAPE, k
    for k in (dict(q_strides=(1, 4)), dict(batch=20000), dict(kv_len=2**30 + 1, capacity=2**31 - 1), dict(q_len=2**21)):
        assert ok(**k) == _ffi.RT_ERR_UNSUPPORTED, k
    for k in (dict(causal=2), dict(scale=float("nan"))):
        assert ok(**k) == _ffi.RT_ERR_INVALID_ARG, k
    assert L.rt_attention_q4_workspace_bytes(ctypes.byref(changed()), None) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_q4_workspace_bytes(ctypes.byref(changed(kv_len=61)), ctypes.byref(need)) == _ffi.RT_ERR_INVALID_SHAPE
    for k in (dict(batch=0), dict(heads=0, kv_heads=0), dict(q_len=0)):
        assert L.rt_attention_q4_workspace_bytes(ctypes.byref(changed(**k)), ctypes.byref(need)) == 0 and need.value == 0
    assert L.rt_attention_q4_enqueue(None, None, None, None, None, None, None, None, None, 0, None) == _ffi.RT_ERR_INVALID_ARG


def test_tensor_guards_without_a_device():
    c = Tensor.empty_cache((2, 3, 20, 48), Device.CPU, DType.Q4_0)
    assert c.is_q4_cache and c.storage.nbytes == cache_q4_nbytes((2, 3, 20, 48))[0]
    h = lambda *s, dt=np.float16: Tensor.from_data(np.zeros(s, dt))
    assert c.cache_write(h(2, 3, 4, 48), 16).shape == c.shape and c.cache_write(h(2, 4, 144), 16).shape == c.shape
    assert c.cache_write(h(2, 4, 144, dt=np.float32), 0).is_q4_cache
    q = h(2, 5, 6 * 48)
    a = q.attention(c, c, causal=True, kv_len=20, merge_heads=True)
    assert a.shape == (2, 5, 288) and a.dt == DType.F16
    assert h(2, 6, 5, 48).attention(c, c, mask=h(2, 1, 5, 20)).shape == (2, 6, 5, 48)
    w = Tensor((2, 3, 20, 64), DType.Q4_0, Device.CPU, np.zeros(0, np.uint8))  # a weight of that shape
    for bad, err in ((lambda: c.cache_write(h(2, 3, 5, 48), 16), InvariantError), (lambda: c.cache_write(h(2, 3, 1, 48), 21), InvariantError),
                     (lambda: c.cache_write(h(2, 3, 1, 48), -1), InvariantError), (lambda: c.cache_write(h(2, 2, 1, 48), 0), OperationError),
                     (lambda: w.cache_write(h(2, 3, 1, 64), 0), InvariantError), (lambda: c.cache(h(2, 3, 1, 48), 2, 0), OperationError),
                     (lambda: h(2, 5, 5 * 48).attention(c, c), InvariantError), (lambda: h(2, 6, 5, 32).attention(c, c), OperationError),
                     (lambda: q.attention(c, c, kv_len=21), OperationError), (lambda: q.attention(c, h(2, 3, 20, 48)), InvariantError),
                     (lambda: h(2, 5, 288, dt=np.float32).attention(c, c), InvariantError), (lambda: q.attention(c, c, mask=h(6, 5, 20)), OperationError),
                     (lambda: q.attention(c, c, mask=h(5, 19)), OperationError), (lambda: c.gemm(h(5, 48), None, False, True, True), InvariantError),
                     (lambda: Tensor.empty_cache((2, 3, 20, 40), Device.CPU, DType.Q4_0), OperationError),
                     (lambda: h(2, 3, 5, 48).attention(h(2, 3, 20, 48), h(2, 3, 20, 48), kv_lens=torch.zeros(2, dtype=torch.int32)), OperationError),
                     (lambda: h(2, 3, 20, 48).cache_write(h(2, 3, 5, 48), 0, offsets=torch.zeros(2, dtype=torch.int32)), OperationError)):
        with pytest.raises(err):
            bad()


# ---- the write --------------------------------------------------------------------------------------------------------------


def write(device, caches, srcs, strides, shape, offset, length, offsets=None, values_out=None, dtype=None):
    b, h, cap, d = shape
    p = lambda t: None if t is None else t.data_ptr()
    v = values_out or (None, None)
    return _ffi.lib().rt_cache_write_q4_enqueue(device.ctx, _ffi.RT_F32 if srcs[0].dtype == torch.float32 else _ffi.RT_F16, p(caches[0]), p(srcs[0]), p(caches[1]),
                                                p(srcs[1]), (ctypes.c_int64 * 3)(*strides), p(v[0]), p(v[1]), p(offsets), b, h, cap, offset, length, d,
                                                torch.cuda.current_stream().cuda_stream)


def rows(rng, shape):
    """f16 rows with what the rounding can go wrong at: scales over the whole range, ties between codes, equal magnitudes of both signs, zeros."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-24, 14, shape[:-1]))[..., None]
    pick = rng.random(shape[:-1])
    x[pick < 0.2] = np.round(x[pick < 0.2] * 4) / 4  # few significant bits: quotients half way between codes
    whole = rng.integers(-16, 17, shape) * 0.5
    x[pick > 0.8] = whole[pick > 0.8]
    x[(pick > 0.5) & (pick < 0.52)] = 0
    with np.errstate(over="ignore"):
        x = x.astype(np.float16)
    return np.where(np.isfinite(x), x, np.float16(65504))


@gpu
@pytest.mark.parametrize("d", DIMS)
def test_write_bytes_and_values(device, d):
    rng = np.random.default_rng(d)
    for b, h, cap, offset, n in [(1, 1, 1, 0, 1), (2, 3, 70, 5, 64), (3, 2, 40, 39, 1), (1, 4, 300, 0, 300), (2, 2, 9, 4, 0), (1, 2, 2100, 50, 2049)]:
        shape = (b, h, cap, d)
        k, v = rows(rng, (b, h, n, d)), rows(rng, (b, h, n, d))
        before = rng.integers(0, 256, cache_q4_nbytes(shape)[0], dtype=np.uint8)
        for inside in (False, True):  # [b, h, n, d] and, as a projection leaves it, [b, n, h * d]
            srcs = [torch.from_numpy(np.ascontiguousarray(x.swapaxes(1, 2)) if inside else x).to("cuda:0") for x in (k, v)]
            strides = [n * h * d, d, h * d] if inside else [h * n * d, n * d, d]
            caches = [torch.from_numpy(before.copy()).to("cuda:0") for _ in range(2)]
            vals = [torch.full((b, h, n, d), float("nan"), dtype=torch.float16, device="cuda:0") for _ in range(2)]
            assert write(device, caches, srcs, strides, shape, offset, n, values_out=vals) == 0
            for x, c, val in zip((k, v), caches, vals):
                codes, ds, want = held(x)
                assert np.array_equal(val.cpu().numpy().astype(np.float64), want)
                exp = before.copy()
                at = cache_q4_nbytes(shape)[1]
                exp[: b * h * cap * d // 2].reshape(b, h, cap, d // 2)[:, :, offset : offset + n] = packed(codes)
                sc = exp[at : at + b * h * cap * scales(d) * 2].view(np.float16).reshape(b, h, cap, scales(d))
                sc[:, :, offset : offset + n] = 0
                sc[:, :, offset : offset + n, : blocks(d)] = ds
                got, zero = c.cpu().numpy(), lambda y: np.where(y[at:].view(np.uint16) == 0x8000, 0, y[at:].view(np.uint16))  # (a scale of -0 is one of 0)
                assert np.array_equal(got[:at], exp[:at]) and np.array_equal(zero(got), zero(exp))


@gpu
def test_write_of_f32_one_tensor_and_not_finite(device):
    rng = np.random.default_rng(3)
    shape, n = (1, 2, 12, 80), 7
    x = (rng.standard_normal((1, 2, n, 80)) * 3).astype(np.float32)
    x[0, 0, 1, 5], x[0, 1, 2, 40], x[0, 1, 3, 79], x[0, 0, 4, 0] = np.inf, -np.inf, np.nan, 1e6  # (1e6 is infinite in f16)
    x[0, 0, 5, 64:] = 0
    cache, val = torch.zeros(cache_q4_nbytes(shape)[0], dtype=torch.uint8, device="cuda:0"), torch.zeros((1, 2, n, 80), dtype=torch.float16, device="cuda:0")
    assert write(device, (cache, None), (torch.from_numpy(x).to("cuda:0"), None), [2 * n * 80, n * 80, 80], shape, 2, n, values_out=(val, None)) == 0
    with np.errstate(over="ignore"):
        codes, ds, want = held(x.astype(np.float16))
    assert np.array_equal(val.cpu().numpy().astype(np.float64), want, equal_nan=True)
    assert np.isnan(want).sum() == 32 * 3 + 16
    all_codes, all_ds = np.zeros(shape, np.uint8), np.zeros((1, 2, 12, 3), np.float16)
    all_codes[:, :, 2:9], all_ds[:, :, 2:9] = codes, ds
    got, exp = cache.cpu().numpy(), buffer(all_codes, all_ds)
    at = cache_q4_nbytes(shape)[1]
    assert np.array_equal(got[:at], exp[:at]) and np.array_equal(got[at:].view(np.float16), exp[at:].view(np.float16), equal_nan=True)


@gpu
def test_write_with_an_offset_per_sequence(device):
    rng = np.random.default_rng(4)
    shape, n = (4, 2, 10, 64), 3
    x = rows(rng, (4, 2, n, 64))
    src = torch.from_numpy(x).to("cuda:0")
    caches = [torch.full((cache_q4_nbytes(shape)[0],), 0xA5, dtype=torch.uint8, device="cuda:0") for _ in range(2)]
    offs = torch.tensor([0, 5, 8, -4], dtype=torch.int32, device="cuda:0")  # + 1: rows 1.., 6.., 9 and two beyond, -3.. and none
    assert write(device, caches, (src, src), [2 * n * 64, n * 64, 64], shape, 1, n, offsets=offs) == 0
    codes, _, _ = held(x)
    want = np.full((4, 2, 10, 32), 0xA5, np.uint8)
    for b, at in enumerate([1, 6, 9, -3]):
        for i in range(n):
            if 0 <= at + i < 10:
                want[b, :, at + i] = packed(codes)[b, :, i]
    for c in caches:
        assert np.array_equal(c.cpu().numpy()[: want.size].reshape(want.shape), want)


@gpu
def test_write_refusals(device):
    shape, n = (1, 2, 8, 64), 4
    c = torch.zeros(cache_q4_nbytes(shape)[0], dtype=torch.uint8, device="cuda:0")
    x = torch.zeros((1, 2, n, 64), dtype=torch.float16, device="cuda:0")
    st = [2 * n * 64, n * 64, 64]
    ok = dict(caches=(c, c), srcs=(x, x), strides=st, shape=shape, offset=0, length=n)
    for change, want in ((dict(offset=5), _ffi.RT_ERR_INVALID_SHAPE), (dict(offset=-1), _ffi.RT_ERR_INVALID_SHAPE), (dict(length=9), _ffi.RT_ERR_INVALID_SHAPE),
                         (dict(shape=(1, 2, 8, 72)), _ffi.RT_ERR_INVALID_SHAPE), (dict(shape=(1, 2, 8, 256)), _ffi.RT_ERR_INVALID_SHAPE),
                         (dict(strides=[0, 4, 64]), _ffi.RT_ERR_UNSUPPORTED), (dict(strides=[-8, 64, 64]), _ffi.RT_ERR_UNSUPPORTED),
                         (dict(caches=(None, c)), _ffi.RT_ERR_INVALID_ARG), (dict(caches=(c, None)), _ffi.RT_ERR_INVALID_ARG),
                         (dict(srcs=(x, None)), _ffi.RT_ERR_INVALID_ARG), (dict(srcs=(x.view(-1)[1:], x)), _ffi.RT_ERR_INVALID_ARG)):
        assert write(device, **{**ok, **change}) == want, change
    assert write(device, **ok) == 0 and write(device, **{**ok, "length": 0}) == 0


# ---- the attention -------------------------------------------------------------------------------------------------------------


def reference(q, kv, vv, scale, mask=None, causal=False, lens=None):
    """q [b, h, lq, d] f16, values kv, vv [b, kv_heads, n, d] -> (out, tolerance) float64."""
    b, h, lq, d = q.shape
    g, n = h // kv.shape[1], kv.shape[2]
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.float64)).to("cuda:0")
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for i in range(b):
        m = n if lens is None else int(min(max(lens[i], 0), n))
        for x in range(h):
            Q, K, V = to(q[i, x]), to(kv[i, x // g, :m]), to(vv[i, x // g, :m])
            s = Q @ K.T.contiguous() * scale
            e = (Q.abs() @ K.abs().T.contiguous() * abs(scale)) * (d / 32 + 36) * 2.0**-23 + s.abs() * 2.0**-22
            if mask is not None:
                M = to((mask if mask.ndim == 2 else mask[i])[:, :m])
                hid = M == -np.inf
                s, e = torch.where(hid, -np.inf, s + torch.where(hid, 0, M)), e + torch.where(hid, 0, M.abs()) * 2.0**-22
            if causal:
                hidden = torch.arange(m, device="cuda:0")[None, :] > torch.arange(lq, device="cuda:0")[:, None] + (m - lq)
                s = s.masked_fill(hidden, -np.inf)
            if m == 0:
                continue
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            l = p.sum(-1, keepdim=True)
            w = p / l
            V0 = torch.where(torch.isfinite(V), V, 0)
            seen = (s > -np.inf).double()
            o = w @ V0
            if not bool(torch.isfinite(V).all()):
                o = torch.where((seen @ (~torch.isfinite(V)).double()) > 0, np.nan, o)
            err = ((2.0**-11 + 2.0**-20) * w + 2 * w * torch.where(seen > 0, e, 0)) @ V0.abs() + 2.0**-25 * (seen @ V0.abs()) / l
            out[i, x], tol[i, x] = o.cpu().numpy(), (err + 2.0**-11 * o.abs() + 2.0**-25).cpu().numpy()
    return out, tol


def drawn_cache(rng, b, kv, cap, d, garbage_from=None):
    """Codes, scales of eight significant bits, values; rows from `garbage_from` on hold anything, NaN scales among it."""
    codes = rng.integers(0, 16, (b, kv, cap, d), dtype=np.uint8)
    ds = (rng.integers(128, 256, (b, kv, cap, blocks(d))) * rng.choice([-1, 1], (b, kv, cap, blocks(d))) / 1024.0).astype(np.float16)
    val = values(codes, ds)
    if garbage_from is not None:
        ds[:, :, garbage_from:] = np.nan
    return buffer(codes, ds), val


def run(device, q, kbuf, vbuf, kv, cap, kv_len, scale=None, mask=None, causal=False, lens=None, workspace=True, heads_inside=True):
    b, h, lq, d = q.shape
    desc = attention_desc(b, h, kv, lq, kv_len, d, cap, int(causal), scale, mask, heads_inside)
    need = ctypes.c_uint64()
    L = _ffi.lib()
    assert L.rt_attention_q4_workspace_bytes(ctypes.byref(desc), ctypes.byref(need)) == 0
    ws = torch.full((need.value + 64,), 0xFF, dtype=torch.uint8, device="cuda:0") if workspace and need.value else None
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to("cuda:0")
    qt, kt, vt = to(q.swapaxes(1, 2) if heads_inside else q), to(kbuf), to(vbuf)
    mt, lt = None if mask is None else to(mask), None if lens is None else to(np.asarray(lens, np.int32))
    out = torch.full((q.size + 8,), float("nan"), dtype=torch.float16, device="cuda:0")
    out[q.size :] = 7
    p = lambda t: None if t is None else t.data_ptr()
    st = L.rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), p(qt), p(kt), p(vt), p(mt), p(lt), p(out), p(ws), need.value if ws is not None else 0,
                                   torch.cuda.current_stream().cuda_stream)
    assert st == 0, L.rt_last_error(device.ctx)
    if ws is not None:
        assert (ws[need.value :] == 0xFF).all()
    assert (out[q.size :] == 7).all()
    got = out[: q.size].cpu().numpy()
    return got.reshape(b, lq, h, d).swapaxes(1, 2) if heads_inside else got.reshape(b, h, lq, d)


def check(got, want, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (int(np.isnan(got).sum()), int(np.isnan(want).sum()))
    bad = ~(np.isnan(want) | (np.abs(got - want) <= tol))
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:4])


# (batch, heads, kv_heads, query rows, keys, capacity)
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 2, 2, 1, 63, 64), (2, 4, 4, 1, 64, 64), (1, 3, 3, 1, 65, 70), (2, 8, 2, 1, 200, 200), (1, 8, 1, 1, 600, 601), (1, 32, 8, 1, 1500, 1600),
          (3, 5, 1, 1, 130, 130), (1, 4, 4, 2, 77, 80), (2, 6, 2, 4, 513, 520), (1, 4, 2, 7, 300, 300), (1, 16, 1, 1, 1025, 1030), (1, 2, 2, 17, 100, 100),
          (2, 4, 2, 9, 257, 260), (1, 2, 1, 70, 333, 333), (1, 4, 4, 130, 130, 140), (1, 1, 1, 33, 20, 20)]


@gpu
@pytest.mark.parametrize("d", DIMS)
def test_attention_shapes(device, d):
    rng = np.random.default_rng(d)
    for b, h, kv, lq, n, cap in SHAPES if d in (80, 128) else SHAPES[1::3] + SHAPES[2::3]:
        kbuf, kval = drawn_cache(rng, b, kv, cap, d, garbage_from=n)
        vbuf, vval = drawn_cache(rng, b, kv, cap, d, garbage_from=n)
        q = rng.standard_normal((b, h, lq, d)).astype(np.float16)
        scale = 1 / np.sqrt(np.float32(d))
        for causal in (False, True):
            want, tol = reference(q, kval[:, :, :n], vval[:, :, :n], float(scale), causal=causal)
            for ws in (True, False):
                check(run(device, q, kbuf, vbuf, kv, cap, n, scale, causal=causal, workspace=ws, heads_inside=ws), want, tol)


@gpu
@pytest.mark.parametrize("lq,causal", [(1, False), (1, True), (3, True), (20, True), (40, False)])
def test_attention_lengths(device, lq, causal):
    """Sequences of their own lengths: none, one, shorter than the queries, out of range; garbage behind each."""
    rng = np.random.default_rng(lq)
    lens = [0, 1, 2, 64, 65, 700, 699, 900, -5]
    b, kv, g, cap, n, d = len(lens), 2, 2, 710, 700, 80
    kbuf, kval = drawn_cache(rng, b, kv, cap, d)
    vbuf, vval = drawn_cache(rng, b, kv, cap, d)
    q = rng.standard_normal((b, kv * g, lq, d)).astype(np.float16)
    want, tol = reference(q, kval[:, :, :n], vval[:, :, :n], 0.125, causal=causal, lens=lens)
    for ws in (True, False):
        check(run(device, q, kbuf, vbuf, kv, cap, n, 0.125, causal=causal, lens=lens, workspace=ws), want, tol)


@gpu
@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("lq", [1, 5, 33])
def test_attention_masks(device, dt, lq):
    """Zeros and -inf, numbers, the type's lowest value, a row that hides everything (NaN), one key left; shared and per sequence."""
    rng = np.random.default_rng(lq)
    b, h, kv, n, d = 2, 4, 2, 205, 64
    kbuf, kval = drawn_cache(rng, b, kv, n, d)
    vbuf, vval = drawn_cache(rng, b, kv, n, d)
    q = rng.standard_normal((b, h, lq, d)).astype(np.float16)
    low = np.finfo(dt).min
    for shape in ((lq, n), (b, lq, n)):
        plain = np.where(rng.random(shape) < 0.4, -np.inf, 0).astype(dt)
        numbers = rng.uniform(-3, 3, shape).astype(dt)
        lowest = np.where(rng.random(shape) < 0.5, low, 0).astype(dt)
        one = np.full(shape, -np.inf, dt)
        one[..., 77] = -1
        none = numbers.copy()
        none[..., 0, :] = -np.inf
        for mask in (plain, numbers, lowest, one, none):
            want, tol = reference(q, kval, vval, 0.125, mask=mask)
            for causal in (False, True) if mask is numbers and lq > 1 else (False,):
                if causal:
                    want, tol = reference(q, kval, vval, 0.125, mask=mask, causal=True)
                check(run(device, q, kbuf, vbuf, kv, n, n, 0.125, mask=mask, causal=causal), want, tol)
        everything = np.full(shape, low, dt)  # all the same: scores below the lowest value's place in f32 vanish with F32 masks
        got = run(device, q, kbuf, vbuf, kv, n, n, 0.0, mask=everything)
        want, tol = reference(q, kval, vval, 0.0, mask=np.zeros(shape, dt))
        check(got, want, tol)


@gpu
@pytest.mark.parametrize("lq", [1, 6, 40])
def test_attention_scales_that_are_not_finite(device, lq):
    """A NaN scale of a hidden key changes nothing, of a seen one its dimensions (values) or the row (keys)."""
    rng = np.random.default_rng(9)
    b, h, kv, n, d = 1, 4, 2, 150, 80
    codes, ds = rng.integers(0, 16, (b, kv, n, d), dtype=np.uint8), np.full((b, kv, n, 3), 0.125, np.float16)
    kds, vds = ds.copy(), ds.copy()
    kds[0, 0, 33, 1] = np.nan   # hidden by the mask
    vds[0, 0, 33, 2] = np.inf
    vds[0, 1, 100, 2] = np.nan  # seen: dimensions 64 .. 79 of the second pair of heads
    vds[0, 1, 33] = np.nan
    mask = np.zeros((lq, n), np.float16)
    mask[:, 33] = -np.inf
    q = rng.standard_normal((b, h, lq, d)).astype(np.float16)
    kval = values(codes, np.where(np.isfinite(kds), kds, 0))
    vval = values(codes, vds)
    vval[0, 0, 33, 64:] = np.nan
    want, tol = reference(q, kval, vval, 0.1, mask=mask)
    assert np.isnan(want[0, 2:, :, 64:]).all() and np.isfinite(want[0, 2:, :, :64]).all() and np.isfinite(want[0, :2]).all()
    check(run(device, q, buffer(codes, kds), buffer(codes, vds), kv, n, n, 0.1, mask=mask), want, tol)
    kds[0, 0, 20, 0] = np.nan  # seen
    got = run(device, q, buffer(codes, kds), buffer(codes, vds), kv, n, n, 0.1, mask=mask)
    assert np.isnan(got[0, :2]).all() and np.isfinite(got[0, 2:, :, :64]).all()


@gpu
def test_attention_refusals(device):
    rng = np.random.default_rng(1)
    kbuf, _ = drawn_cache(rng, 1, 2, 8, 64)
    buf, q = torch.from_numpy(kbuf).to("cuda:0"), torch.zeros((1, 2, 1, 64), dtype=torch.float16, device="cuda:0")
    L = _ffi.lib()

    def call(desc=None, q_=q.data_ptr(), k=buf.data_ptr(), mask=None, lens=None, out=q.data_ptr()):
        desc = desc or attention_desc(1, 2, 2, 1, 8, 64, 8)
        return L.rt_attention_q4_enqueue(device.ctx, ctypes.byref(desc), q_, k, buf.data_ptr(), mask, lens, out, None, 0, None)

    assert call() == 0
    for kw in (dict(q_=None), dict(k=None), dict(out=None), dict(q_=q.data_ptr() + 2), dict(k=buf.data_ptr() + 8), dict(out=q.data_ptr() + 1), dict(lens=buf.data_ptr() + 2)):
        assert call(**kw) == _ffi.RT_ERR_INVALID_ARG, kw
    d = attention_desc(1, 2, 2, 1, 8, 64, 8)
    assert call(d, mask=buf.data_ptr()) == _ffi.RT_ERR_INVALID_SHAPE  # rows of no stride
    d.mask_strides[1], d.mask_dtype = 8, _ffi.RT_F32
    assert call(d, mask=buf.data_ptr() + 2) == _ffi.RT_ERR_INVALID_ARG
    d.mask_dtype = _ffi.RT_Q4_0
    assert call(d, mask=buf.data_ptr()) == _ffi.RT_ERR_DTYPE_MISMATCH


# ---- together: the modules on a 4-bit cache ----------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("offsets", [False, True])
def test_decode_steps_through_the_modules(device, offsets):
    """A prompt, then token by token: SelfAttention on a 4-bit KVCache with Q4_0 projections, against float64 over the values the cache holds."""
    from test_q4_0 import draw, segments, values as weight_values
    rng = np.random.default_rng(11)
    H, D, cap, steps = 4, 48, 40, [9, 1, 1, 3, 1]
    W = H * D
    lin, ws = [], []
    for i in range(4):
        codes, d = draw(W * W, i)
        d = (d.astype(np.float32) * 0.5).astype(np.float16)
        ws.append(weight_values(codes, d).reshape(W, W))
        lin.append(nn.Linear(Tensor.from_quantized(segments(codes, d), DType.Q4_0, (W, W), device)))
    attn = nn.SelfAttention(*lin, H)
    cache = nn.KVCache(1, (1, H, cap, D), device, DType.Q4_0)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    kall, vall = np.zeros((1, H, 0, D)), np.zeros((1, H, 0, D))
    for n in steps:
        x = Tensor.from_data((rng.standard_normal((1, n, W)) * 0.3).astype(np.float16), None, device)
        if offsets:  # the same calls one by one, with lengths on the device
            e = cache[0]
            q, k, v = (l.schedule(x) for l in lin[:3])
            off = zero + e.entries
            keys, vals = e.k_cache.cache_write(k, 0, offsets=off), e.v_cache.cache_write(v, 0, offsets=off)
            a = q.attention(keys, vals, causal=True, kv_len=cap, merge_heads=True, kv_lens=off + n)
            got = lin[3].schedule(a).resolve()
        else:
            q, k, v = (l.schedule(x) for l in lin[:3])
            got = attn.schedule(x, cache[0]).resolve()
        split = lambda t: t.resolve().to(Device.CPU).storage.reshape(1, n, H, D).swapaxes(1, 2)
        q, k, v = split(q), split(k), split(v)  # as the projections round them
        kall, vall = np.concatenate([kall, held(k)[2]], 2), np.concatenate([vall, held(v)[2]], 2)
        want, tol = reference(q, kall, vall, 1 / np.sqrt(D), causal=True)
        o = want.swapaxes(1, 2).reshape(n, W)
        to = tol.swapaxes(1, 2).reshape(n, W)
        y, mag = o @ ws[3].T, np.abs(o) @ np.abs(ws[3]).T
        bound = to @ np.abs(ws[3]).T + 2.0**-11 * np.abs(y) + 2.0**-23 * (W / 32 + 56) * mag + 2.0**-25
        g = got.to(Device.CPU).storage.reshape(n, W).astype(np.float64)
        assert (np.abs(g - y) <= bound).all(), float((np.abs(g - y) / bound).max())
        cache.update(n)
    codes = cache[0].k_cache.to(Device.CPU).storage[: H * cap * D // 2].reshape(1, H, cap, D // 2)
    assert not codes[:, :, sum(steps) :].any()  # rows behind the last are as they were
