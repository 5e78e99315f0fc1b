"""Attention over 4-bit caches at the ends of its numbers' range.  Caches and the call are those of test_cache_q4."""
import numpy as np
import pytest

from test_cache_q4 import blocks, buffer, run

gpu = pytest.mark.gpu


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
