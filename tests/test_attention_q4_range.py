"""Attention over 4-bit caches at the ends of its numbers' range.  Caches and the call are those of test_cache_q4."""
import ctypes

import numpy as np
import pytest

from ratchet_amd import _ffi
from test_cache_q4 import attention_desc, blocks, buffer, check, reference, run, values

gpu = pytest.mark.gpu


def test_tiles_of_a_call():
    """A launch has fewer than 2^32 threads along an axis, 2^23 - 1 workgroups of 512, a tile of 128 rows each; up to 16 rows per head of keys take no tiles."""
    L, need = _ffi.lib(), ctypes.c_uint64()
    for batch, kv, heads, lq, want in ((65535, 1, 1, 128 * 128, 0), (65535, 1, 1, 128 * 128 + 1, _ffi.RT_ERR_UNSUPPORTED), (8191, 8, 64, 2048, 0), (8191, 8, 64, 2049, _ffi.RT_ERR_UNSUPPORTED),
                                       (511, 1, 1, 32 * 65535, 0), (512, 1, 1, 32 * 65535, _ffi.RT_ERR_UNSUPPORTED), (65535, 1, 16, 1, 0), (1, 1, 1, 32 * 65535, 0)):
        for n in (1, 1000, 1 << 30):
            d = attention_desc(batch, heads, kv, lq, n, 16, n)
            assert L.rt_attention_q4_validate(ctypes.byref(d)) == want, (batch, kv, lq, n)
            assert L.rt_attention_q4_workspace_bytes(ctypes.byref(d), ctypes.byref(need)) == want
            if want == 0:  # and the shares that a workspace makes are no more, nor the rows that a second launch joins
                tiles, shares = batch * kv * -(-lq * heads // kv // 128), need.value // (batch * heads * lq * 18 * 4)
                assert lq * heads // kv <= 16 or tiles * max(shares, 1) < 1 << 23
                assert not shares or batch * heads * lq <= 1 << 18
    for k in (dict(batch=0), dict(heads=0, kv_heads=0), dict(q_len=0)):
        d = attention_desc(2, 8, 4, 3, 50, 64, 60)
        for name, v in k.items():
            setattr(d, name, v)
        assert L.rt_attention_q4_validate(ctypes.byref(d)) == 0


def one_dimension(n, d, k0, v0, extra=None):
    """A cache whose keys have k0 [n] in dimension 0 (and `extra` in dimension 32), whose values have v0 [n] in every dimension: codes 9, scales the numbers."""
    kc, kd = np.full((1, 1, n, d), 8, np.uint8), np.zeros((1, 1, n, blocks(d)), np.float16)
    kc[..., 0], kd[0, 0, :, 0] = 15, k0
    if extra is not None:
        kc[..., 32], kd[0, 0, :, 1] = 9, extra
    vc, vd = np.full((1, 1, n, d), 9, np.uint8), np.repeat(np.asarray(v0, np.float16)[None, None, :, None], blocks(d), -1)
    return buffer(kc, kd), buffer(vc, vd)


@gpu
@pytest.mark.parametrize("lq", [1, 13, 20, 150])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_past_two_to_the_27(device, lq, sign):
    """Products and sums that f32 holds exactly, and after the scale a rounding of up to 2^6: some keys share the largest, all others are 2^15 such roundings below it.  Their weights
    are 0 in any order of the roundings, so that a row is the mean of the values of the former: exact but for the rounding to f16."""
    n, d = 700, 64
    rng = np.random.default_rng(lq)
    v0 = rng.integers(-64, 65, n) / 16
    k0 = np.full(n, 1024.0 if sign > 0 else 4096.0)  # times 7 and the query's 4096
    best = [3, 200, 201, 640, 699]
    k0[best] = 4096 if sign > 0 else 1024
    kbuf, vbuf = one_dimension(n, d, k0, v0)
    q = np.zeros((1, 1, lq, d), np.float16)
    q[..., 0] = sign * 4096
    for scale in np.float32([1.0, 1.3, 2.0, 3.7, 5.5, 9.0, 11.0, 17.0, 33.0, 100.0]):
        got = run(device, q, kbuf, vbuf, 1, n, n, scale)
        assert (np.abs(got.astype(np.float64) - v0[best].mean()) <= 2.0**-11 * np.abs(v0[best].mean()) + 2.0**-20).all(), (scale, got[0, 0, :, 0])
        mask = np.zeros((lq, n), np.float16)
        mask[:, best[0]] = -np.inf
        got = run(device, q, kbuf, vbuf, 1, n, n, scale, mask=mask)
        assert (np.abs(got.astype(np.float64) - v0[best[1:]].mean()) <= 2.0**-11 * np.abs(v0[best[1:]].mean()) + 2.0**-20).all(), scale


@gpu
@pytest.mark.parametrize("step", [8, 16])
def test_large_scores_a_step_apart(device, step):
    """Scores between 2^27 and 2^28 in base 2, where an f32 moves by 16: later keys are one such step above the first.  What the two weigh is a matter of rounding; a row is a
    mean of the values 1 and 2 in any case."""
    n, d, lq = 512, 64, 160
    kbuf, vbuf = one_dimension(n, d, np.full(n, 4096.0), np.where(np.arange(n) < 256, 1, 2), extra=np.where(np.arange(n) < 256, 0, step))
    for length in (n, n - 5):  # whole blocks, and a last one that is not
        for base in range(3264, 4600, 160):
            q = np.zeros((1, 1, lq, d), np.float16)
            q[0, 0, :, 0] = base + 16 * (np.arange(lq) // 16)  # (rows of a tile move together)
            q[..., 32] = 1
            for ws in (True, False):
                got = run(device, q, kbuf, vbuf, 1, n, length, 1.0, workspace=ws).astype(np.float64)
                assert ((got >= 1 - 2.0**-10) & (got <= 2 + 2.0**-9)).all(), (base, got[0, 0, :, 0])


@gpu
@pytest.mark.parametrize("lq", [1, 6, 13, 17, 40, 150])
@pytest.mark.parametrize("d", [48, 96, 128])
def test_scales_above_what_a_value_can_follow(device, lq, d):
    """8188 is the last scale whose values, up to eight times it, are f16 numbers; from 8192 on a block counts as one that is not finite.  Hidden, by a mask or by the causal flag, it
    changes nothing; seen it leaves other rows alone, and is NaN in its dimensions (values; a row that sees such keys is not defined)."""
    rng = np.random.default_rng(d + lq)
    n = 333
    codes = rng.integers(0, 16, (1, 1, n, d), dtype=np.uint8)
    vcodes = rng.integers(0, 16, (1, 1, n, d), dtype=np.uint8)
    ds = np.full((1, 1, n, blocks(d)), 0.125, np.float16)
    q = rng.standard_normal((1, 1, lq, d)).astype(np.float16)
    q[..., 32:] *= np.float16(0.01)
    mask = rng.uniform(-2, 2, (lq, n)).astype(np.float32)
    hidden = [7, 64, 200, 332]
    mask[:, hidden] = -np.inf
    for big in (16384.0, -8192.0, 65504.0, np.inf):
        kds, vds = ds.copy(), ds.copy()
        kds[0, 0, hidden, 1], vds[0, 0, hidden, 1] = big, big
        codes[0, 0, hidden, 32:], vcodes[0, 0, hidden, 32:] = 0, 0
        plain = lambda c: values(c, ds)
        want, tol = reference(q, plain(codes), plain(vcodes), 0.1, mask=mask)
        for ws in (True, False):
            check(run(device, q, buffer(codes, kds), buffer(vcodes, vds), 1, n, n, 0.1, mask=mask, workspace=ws), want, tol)
        # seen, by the last row alone
        open_ = mask.copy()
        open_[lq - 1, 200] = 0
        got = run(device, q, buffer(codes, kds), buffer(vcodes, ds), 1, n, n, 0.1, mask=open_)
        check(got[:, :, : lq - 1], *(x[:, :, : lq - 1] for x in reference(q, plain(codes), plain(vcodes), 0.1, mask=open_)))
        got = run(device, q, buffer(codes, ds), buffer(vcodes, vds), 1, n, n, 0.1, mask=open_)
        assert np.isnan(got[0, 0, lq - 1, 32:64]).all() and np.isfinite(got[0, 0, lq - 1, :32]).all() and np.isfinite(got[0, 0, lq - 1, 64:]).all(), big
        # the last key is seen by the last row alone
        kds, vds = ds.copy(), ds.copy()
        kds[0, 0, n - 1, 1], vds[0, 0, n - 1, 1] = big, big
        want, tol = (x[:, :, : lq - 1] for x in reference(q, plain(codes), plain(vcodes), 0.1, causal=True))
        check(run(device, q, buffer(codes, kds), buffer(vcodes, vds), 1, n, n, 0.1, causal=True)[:, :, : lq - 1], want, tol)
        got = run(device, q, buffer(codes, ds), buffer(vcodes, vds), 1, n, n, 0.1, causal=True)
        assert np.isnan(got[0, 0, lq - 1, 32:64]).all()
        check(got[:, :, : lq - 1], want, tol)
    # 8188: values up to 65504, all of them f16 numbers
    kds, vds = ds.copy(), ds.copy()
    kds[0, 0, 200, 1] = vds[0, 0, 200, 1] = 8188
    codes[0, 0, 200, 32:64] = 8
    codes[0, 0, 200, 32], vcodes[0, 0, 200, 32:64] = 0, rng.integers(0, 2, min(d, 64) - 32) * 15
    q[..., 32] = np.float16(2.0**-14)  # a score of -4
    want, tol = reference(q, values(codes, kds), values(vcodes, vds), 0.1)
    check(run(device, q, buffer(codes, kds), buffer(vcodes, vds), 1, n, n, 0.1), want, tol)


@gpu
@pytest.mark.parametrize("lq", [1, 6, 13, 17, 150])
@pytest.mark.parametrize("masked", [False, True])
def test_a_long_tail_beside_one_large_probability(device, lq, masked):
    """One key 25.5 powers of two above 2^16 others, that weigh 2^-9.5 together and, since its value is 0, are all that a row consists of.  As f16 numbers
    relative to the largest they would be lost: what a probability is rounded to, 2^-25 of the largest at least, is more than they are.  With one workgroup, and so on the keys of one wavefront in eight
    (one half of them), or with shares.  Tolerance: as in test_cache_q4, but for its 2^-25 sum_j |v| / l, which is 2^-32 here: a probability of the largest is held at 2^7 or more of f16."""
    n, d = 1 << 16, 32
    rng = np.random.default_rng(lq)
    kc, kd = np.full((1, 1, n, d), 8, np.uint8), np.full((1, 1, n, 1), 0.5, np.float16)
    at = 1000
    kc[0, 0, at, 0] = 12  # 2 in dimension 0
    vc, vd = rng.integers(9, 16, (1, 1, n, d), dtype=np.uint8), np.full((1, 1, n, 1), 8.0, np.float16)
    vc[0, 0, at] = 8
    q = np.zeros((1, 1, lq, d), np.float16)
    q[..., 0] = np.linspace(0.99, 1, lq)
    scale = np.float32(25.5 * np.log(2) / 2)
    mask = np.zeros((lq, n), np.float16) if masked else None
    kval, vval = values(kc, kd), values(vc, vd)
    want, tol = reference(q, kval, vval, float(scale), mask=mask)
    s = q[0, 0, :, 0].astype(np.float64) * 2 * float(scale)
    tol -= ((2.0**-25 - 2.0**-32) * vval[0, 0].sum(0)[None] / (1 + n * np.exp(-s))[:, None])[None, None]
    assert (want > 0.01).all() and (tol < 0.02 * want).all()
    for ws in (True, False):
        check(run(device, q, buffer(kc, kd), buffer(vc, vd), 1, n, n, scale, mask=mask, workspace=ws), want, tol)


@gpu
@pytest.mark.parametrize("lq", [1, 6, 13, 20, 150])
@pytest.mark.parametrize("near", [0.999, 0.9, 0.72, 0.5])
def test_masks_near_the_lowest_number(device, lq, near):
    """A mask of f32's lowest number and a few keys above it by a part of that: differences of 10^35 and more, so that a row is the mean of the values of those few (next to such a mask
    their scores vanish in f32).  They lie in one block of 64 keys, in two of them, or at both ends."""
    n, d = 1500, 64
    rng = np.random.default_rng(lq)
    v0 = rng.integers(-64, 65, n) / 16
    kbuf, vbuf = one_dimension(n, d, rng.uniform(-0.1, 0.1, n), v0)
    q = rng.standard_normal((1, 1, lq, d)).astype(np.float16)
    low = np.finfo(np.float32).min
    for best in ([70, 71], [3, 700], [0, 1499], [1490]):
        mask = np.full((lq, n), low, np.float32)
        mask[:, best] = np.float32(near * float(low))
        want = v0[best].mean()
        for ws in (True, False):
            got = run(device, q, kbuf, vbuf, 1, n, n, 0.125, mask=mask, workspace=ws).astype(np.float64)
            assert (np.abs(got - want) <= 2.0**-11 * abs(want) + 2.0**-20).all(), (best, ws, got[0, 0, :, 0], want)
    mask[:] = low  # all alike: the mean of all, each probability and the sum of them rounded
    for ws in (True, False):
        got = run(device, q, kbuf, vbuf, 1, n, n, 0.125, mask=mask, workspace=ws).astype(np.float64)
        assert (np.abs(got - v0.mean()) <= 2.0**-11 * abs(v0.mean()) + 2.0**-11 * np.abs(v0).mean()).all()
