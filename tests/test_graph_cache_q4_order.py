"""The two writes of an attention into 4-bit caches share a launch only where their order cannot matter.  On the CPU a library that writes host memory, a value row before
each key row as the two halves of a launch may, stands in for the device; on the GPU what the lazy graph leaves is compared with one node after the other."""
import ctypes

import numpy as np
import pytest
import torch

import ratchet_amd.tensor as mirror
from ratchet_amd import Device, DType, Tensor
from test_cache_q4 import cache_tensor, drawn_cache

H, CAP, D = 2, 8, 32
ROWS = H * CAP * D // 2  # bytes of a cache's codes


class HostLibrary:
    """rt_cache_write_q4_enqueue for [1, H, CAP, D]: a row's codes are the first bytes of its source, which is enough to tell orders apart."""

    def __init__(self):
        self.pairs = self.calls = 0

    @staticmethod
    def write(cache, src, size, strides, offset, rows):
        for r in range(rows):
            for h in range(H):
                yield lambda r=r, h=h: ctypes.memmove(cache + D // 2 * (h * CAP + offset + r), src + size * (h * strides[1] + r * strides[2]), D // 2)

    def rt_cache_write_q4_enqueue(self, ctx, dt, kc, ks, vc, vs, strides, kv, vv, offsets, batch, heads, capacity, offset, rows, head_dim, stream):
        self.calls += 1
        assert (heads, capacity, head_dim, kv, vv) == (H, CAP, D, None, None)
        if offsets is not None:
            offset += ctypes.cast(offsets, ctypes.POINTER(ctypes.c_int32))[0]
        size = 4 if dt == DType.F32 else 2
        keys = self.write(kc, ks, size, strides, offset, rows)
        if vc is None:
            for step in keys:
                step()
            return 0
        self.pairs += 1
        for a, b in zip(self.write(vc, vs, size, strides, offset, rows), keys):
            a(), b()
        return 0


def arrange(name, cache, source):
    """The keys' and the values' write, and the memory that both leave behind."""
    gen = torch.Generator().manual_seed(7)
    rows = lambda n=4, dt=torch.float16: torch.randn((1, H, n, D), generator=gen).to(dt)
    fresh = lambda: torch.randint(0, 256, (ROWS + 256,), generator=gen, dtype=torch.uint8)
    km, vm, k, v = fresh(), fresh(), rows(), rows()
    KC, VC, keys, values, at = cache(km), cache(vm), source(k), source(v), [0, 0]
    over = lambda m: source(m[: H * 4 * D * 2].view(torch.float16).view(1, H, 4, D))  # halves of a cache's own bytes
    offsets = None, None
    if name == "values are the key cache's bytes":
        values = over(km)
    if name == "keys are the value cache's bytes":
        keys = over(vm)
    if name == "one memory for both":
        VC = cache(km)
    if name == "memories that overlap":
        both = torch.cat([fresh(), fresh()])[: ROWS + 256 + D]
        km, vm = both[: ROWS + 256], both[D:]
        KC, VC = cache(km), cache(vm)
    if name == "sources of two types":
        values = source(rows(dt=torch.float32))
    if name == "sources of f32":
        keys, values = source(rows(dt=torch.float32)), source(rows(dt=torch.float32))
    if name == "other offsets":
        at = [0, 3]
    if name == "other lengths":
        values = source(rows(3))
    one = torch.tensor([2], dtype=torch.int32)
    if name == "offsets in one tensor":
        offsets = one, one
    if name == "offsets in two tensors":
        offsets = one, torch.tensor([3], dtype=torch.int32)
    if name == "offsets of one":
        offsets = one, None
    if name == "the keys written twice":
        KC = KC.cache_write(source(rows()), 0)
    return KC.cache_write(keys, at[0], offsets[0]), VC.cache_write(values, at[1], offsets[1]), (km, vm)


@pytest.mark.parametrize("name", ["apart", "sources of f32", "offsets in one tensor", "values are the key cache's bytes", "keys are the value cache's bytes", "one memory for both",
                                  "memories that overlap", "sources of two types", "other offsets", "other lengths", "offsets in two tensors", "offsets of one",
                                  "the keys written twice"])
def test_order_of_the_writes(monkeypatch, name):
    device = Device("gpu")
    device._ctx, device._torch_device = object(), torch.device("cpu")
    library = HostLibrary()
    monkeypatch.setattr(mirror._ffi, "lib", lambda: library)

    def cache(m):
        t = Tensor((1, H, CAP, D), DType.Q4_0, device, m)
        t.is_q4_cache = True
        return t

    source = lambda t: Tensor(tuple(t.shape), DType.F32 if t.dtype == torch.float32 else DType.F16, device, t.view(torch.uint8).reshape(-1))
    left = []
    for pair in (False, True):
        k, v, memory = arrange(name, cache, source)
        if pair:
            mirror._write_key_and_value(k, v, 0)
        for t in (k, v):
            if t.storage is None:
                t._execute(0)
        left.append([m.clone() for m in memory])
    assert library.pairs == (name in ("apart", "sources of f32", "offsets in one tensor"))
    assert library.calls == 4 - library.pairs + 2 * (name == "the keys written twice")
    assert all(torch.equal(a, b) for a, b in zip(*left))


@pytest.mark.gpu
@pytest.mark.parametrize("reader", ["nobody", "queries", "values", "values from the key cache as it was", "the keys of both"])
def test_what_reads_the_caches_between_the_writes(device, reader):
    """Queries or values that are themselves an attention over these caches, before the writes or between them."""
    rng = np.random.default_rng(5)
    h, n, d = 2, 16, 64
    start = [drawn_cache(rng, 1, h, n, d)[0] for _ in range(2)]
    rows = [rng.standard_normal((1, h, n, d)).astype(np.float16) for _ in range(5)]

    def attend(lazy):
        step = (lambda t: t) if lazy else (lambda t: t.resolve())
        KC, VC = (cache_tensor(b.copy(), (1, h, n, d), device) for b in start)
        q, k1, k2, v1, v2 = (Tensor.from_data(x, None, device) for x in rows)
        if reader == "queries":
            q = step(q.attention(step(KC.cache_write(k1, 0)), step(VC.cache_write(v1, 0))))
        if reader == "values from the key cache as it was":
            v2 = q.attention(KC, KC).resolve()
        written = step(KC.cache_write(k2, 0))
        if reader == "values":
            v2 = step(q.attention(written, written))
        if reader == "the keys of both":
            k2 = v2
            written = step(KC.cache_write(k2, 0))
        out = q.attention(written, step(VC.cache_write(v2, 0)), causal=True).resolve()
        return [t.to(Device.CPU).storage.copy() for t in (out, KC, VC)]

    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(attend(True), attend(False)))
