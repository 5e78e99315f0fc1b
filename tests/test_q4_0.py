"""Q4_0: the segment layout, the GGUF blocks and their transcoding, and the products with Q4_0 weights, against float64.

The weights of a test are drawn as codes and scales and written into both layouts here, from their definitions: a value is d * (code - 8); a GGUF block
is {f16 d; qs[16]} with values j and j + 16 in byte j; a segment dword holds eight codes, the even values' in nibbles 0..3, the odd ones' in 4..7.

Tolerance of a product: one f16 rounding, at most 2^-11 of the value (2^-25 below the normal range), and the f32 sums'.  Codes and activations enter the
matrix cores exactly; a block's sum has 32 terms, then K / 32 scaled sums and at most 24 partial ones (wavefronts, shares of K, the bias) are added:
K / 32 + 56 roundings of partial sums that never exceed sum |w| |x| + |bias|, 2^-23 each with the matrix cores' own order and truncation allowed for."""
import ctypes
import struct

import numpy as np
import pytest
import torch

from ratchet_amd import DType, Device, InvariantError, OperationError, Tensor, _ffi, dequantize, gguf, tensor_nbytes, transcode_gguf_q4_0
from ratchet_amd.tensor import Matmul

gpu = pytest.mark.gpu


def draw(numel, seed):
    """(codes 0..15, f16 scales): every code, scales of either sign, zeros and subnormals among them."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, numel, dtype=np.uint8)
    d = (rng.uniform(0.3, 2.0, numel // 32) * rng.choice([-1, 1], numel // 32) / 64).astype(np.float16)
    d[rng.random(len(d)) < 0.03] = 0
    d[rng.random(len(d)) < 0.03] = np.float16(3e-6)
    return codes, d


def values(codes, d):
    return (codes.astype(np.float64).reshape(-1, 32) - 8) * d.astype(np.float64)[:, None]


def padded(b):
    return np.concatenate([b, np.zeros(-len(b) % 256, np.uint8)])


def segments(codes, d):
    out = np.zeros(codes.size // 8, np.uint32)
    for e in range(8):
        out |= codes.reshape(-1, 8)[:, e].astype(np.uint32) << np.uint32(4 * (e // 2 + 4 * (e % 2)))
    return np.concatenate([padded(out.view(np.uint8)), padded(d.view(np.uint8))])


def gguf_blocks(codes, d):
    c = codes.reshape(-1, 32)
    return np.concatenate([d.view(np.uint8).reshape(-1, 2), c[:, :16] | c[:, 16:] << 4], 1).reshape(-1)


# ---- on the CPU --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("numel", [0, 32, 256, 512, 544, 32 * 8 * 64, 51865 * 32])
def test_sizes(numel):
    codes, d = draw(numel, 1)
    assert tensor_nbytes(DType.Q4_0, numel) == len(segments(codes, d))
    assert _ffi.lib().rt_q4_0_scale_offset(numel) == len(padded(np.zeros(numel // 2, np.uint8)))


def test_refusals_on_the_host():
    L, n = _ffi.lib(), ctypes.c_uint64()
    assert L.rt_tensor_nbytes(_ffi.RT_Q4_0, 40, ctypes.byref(n)) == _ffi.RT_ERR_UNSUPPORTED
    assert L.rt_transcode_gguf_q4_0(None, None, 1, None, None) == _ffi.RT_ERR_INVALID_ARG
    w = lambda shape: Tensor(shape, DType.Q4_0, Device.CPU, np.zeros(0, np.uint8))
    x = lambda shape, dt=DType.F16: Tensor(shape, dt, Device.CPU, np.zeros(0, np.uint8))
    assert w((64, 96)).gemm(x((5, 96)), None, False, True, True).shape == (5, 64)
    assert x((5, 96)).matmul(w((64, 96)), False, True).shape == (5, 64)
    for bad, st in ((lambda: w((64, 40)).gemm(x((5, 40)), None, False, True, True), _ffi.RT_ERR_UNSUPPORTED),       # K is no whole number of blocks
                    (lambda: w((64, 96)).gemm(x((64, 5)), None, True, False, False), _ffi.RT_ERR_UNSUPPORTED),      # transposed weight
                    (lambda: w((64, 96)).gemm(x((5, 96), DType.F32), None, False, True, True), _ffi.RT_ERR_DTYPE_MISMATCH),
                    (lambda: x((5, 64)).matmul(w((64, 96)), False, False), _ffi.RT_ERR_UNSUPPORTED)):
        with pytest.raises((InvariantError, OperationError)) as e:
            bad()
        assert e.value.status == st
    spec = Matmul(w((64, 96)), x((5, 96)), None, False, True, True).compute_spec()
    assert _ffi.lib().rt_kernel_string(spec.kernel) != b"unknown"
    for dt in (_ffi.RT_Q4_0 + 1, -1):
        d = _ffi.make_desc(dt, (64, 96), _ffi.RT_F16, (5, 96), False, True, True)
        assert L.rt_matmul_validate(ctypes.byref(d)) == _ffi.RT_ERR_INVALID_ARG


# ---- on the GPU: formats --------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("numel", [32, 96, 512 * 3, 255 * 32, 257 * 32, 8192 * 32 + 32])
def test_transcode_and_dequantize(device, numel):
    codes, d = draw(numel, numel)
    d[0] = np.float16(65504)
    t = transcode_gguf_q4_0(gguf_blocks(codes, d), (numel,), device)
    assert np.array_equal(t.to(Device.CPU).storage, segments(codes, d))
    got = dequantize(t).to(Device.CPU).storage
    assert np.array_equal(got.reshape(-1).astype(np.float64), values(codes, d).reshape(-1))  # 11 + 4 bits: exact in f32


def image(name, shape, blocks):
    """A GGUF v3 file with one Q4_0 tensor."""
    s = lambda b: struct.pack("<Q", len(b)) + b
    head = b"GGUF" + struct.pack("<IQQ", 3, 1, 0) + s(name) + struct.pack("<I", len(shape)) + b"".join(struct.pack("<Q", v) for v in reversed(shape))
    head += struct.pack("<IQ", 2, 0)
    return head + bytes(-len(head) % 32) + blocks.tobytes()


@gpu
def test_gguf_tensor_through_a_linear(device):
    codes, d = draw(48 * 160, 5)
    head = gguf.Header.read(image(b"blk.0.ffn_up.weight", (48, 160), gguf_blocks(codes, d)))
    with pytest.raises(OperationError):  # as the reference does
        head.tensor("blk.0.ffn_up.weight", device)
    w = head.tensor("blk.0.ffn_up.weight", device, q4_0=True)
    assert w.dt == DType.Q4_0 and w.shape == (48, 160) and np.array_equal(w.to(Device.CPU).storage, segments(codes, d))
    st = _ffi.lib().rt_gguf_load_tensor(device.ctx, head._h, head._buf, len(head._image), 0, _ffi.RT_Q4_0, None, w.data_ptr(), None)
    assert st == _ffi.RT_ERR_INVALID_ARG  # no staging buffer
    st = _ffi.lib().rt_gguf_load_tensor(device.ctx, head._h, head._buf, len(head._image), 0, _ffi.RT_Q8_0H, w.data_ptr(), w.data_ptr(), None)
    assert st == _ffi.RT_ERR_UNSUPPORTED
    from ratchet_amd import nn
    x = np.random.default_rng(2).standard_normal((1, 3, 160)).astype(np.float16)
    y = nn.Linear(w).schedule(Tensor.from_data(x, None, device)).resolve().to(Device.CPU).storage
    W = values(codes, d).reshape(48, 160)
    check(y.reshape(3, 48), x[0].astype(np.float64) @ W.T, np.abs(x[0].astype(np.float64)) @ np.abs(W).T, 160)


# ---- on the GPU: products ----------------------------------------------------------------------------------------------------


def check(got, want, mag, k, slope=1.0, rel=0.0):
    got = torch.as_tensor(got).double().cpu().numpy()
    tol = (2.0**-11 + rel) * np.abs(want) + slope * 2.0**-23 * (k / 32 + 56) * mag + 2.0**-25
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / tol).max()), np.argwhere(bad)[:3])


def operands(device, stack, m, k, n, seed=0):
    rng = np.random.default_rng(m * 7 + k * 3 + n + seed)
    s = stack[0] if stack else 1
    codes, d = draw(s * m * k, m + k + n)
    w = values(codes, d).reshape(s, m, k)
    x = rng.standard_normal((s, n, k)).astype(np.float16)
    x[0, 0, ::7] *= np.float16(50)
    bias = [rng.standard_normal(v).astype(np.float16) for v in (m, n)]
    weight = Tensor.from_quantized(segments(codes, d), DType.Q4_0, (*stack, m, k), device)
    W, X = (torch.from_numpy(v.astype(np.float64)).to("cuda:0") for v in (w, x))
    want = torch.stack([X[i] @ W[i].T for i in range(s)]).cpu().numpy()
    mag = torch.stack([X[i].abs() @ W[i].abs().T for i in range(s)]).cpu().numpy()
    return weight, x.reshape(*stack, n, k), bias, want, mag


# (stack, weight rows, K, activation rows): one of everything, ends inside every tile, each number of vectors that has a rule, K of one to many
# blocks and of no whole number of larger units, one wavefront's share of K empty, many rows
SIZES = [((), 1, 32, 1), ((), 5, 64, 2), ((), 16, 96, 1), ((), 17, 128, 3), ((), 33, 160, 4), ((), 100, 224, 5), ((), 257, 256, 8), ((), 130, 480, 9),
         ((), 64, 512, 16), ((), 1000, 736, 17), ((), 31, 1024, 31), ((), 515, 1280, 33), ((), 48, 2560, 48), ((), 49, 2592, 64), ((), 200, 384, 65),
         ((), 2561, 2560, 1), ((), 300, 10240, 1), ((), 300, 10240, 4), ((), 160, 11008, 13), ((), 51865, 384, 1), ((), 51865, 256, 7),
         ((), 320, 768, 130), ((), 161, 2560, 300), ((), 1024, 1056, 129), ((3,), 40, 288, 1), ((3,), 40, 256, 20), ((2,), 170, 512, 100), ((), 640, 5120, 512)]


@gpu
@pytest.mark.parametrize("stack,m,k,n", SIZES)
def test_products(device, stack, m, k, n):
    weight, x, bias, exact, mag = operands(device, stack, m, k, n)
    s = stack[0] if stack else 1
    xt = Tensor.from_data(x, None, device)
    for to in (True, False):
        for b in (bias[0 if to else 1], None):
            got = weight.gemm(xt, None if b is None else Tensor.from_data(b, None, device), False, True, to).resolve().to(Device.CPU).storage
            got = got.reshape(s, n, m) if to else got.reshape(s, m, n).swapaxes(1, 2)
            off = 0 if b is None else b.astype(np.float64) if to else b.astype(np.float64)[:, None]
            check(got, exact + off, mag + np.abs(off), k)


@gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(100, 256, 1), (259, 2560, 5), (64, 96, 20), (320, 512, 200)])
def test_activation_behind_a_product(device, act, m, k, n):
    weight, x, bias, exact, mag = operands(device, (), m, k, n)
    y = exact[0] + bias[0].astype(np.float64)
    got = getattr(weight.gemm(Tensor.from_data(x, None, device), Tensor.from_data(bias[0], None, device), False, True, True), act)()
    got = got.resolve().to(Device.CPU).storage
    z = y if act == "silu" else 2 * y * (0.035677407 * y * y + 0.7978846)
    # |slope| <= 1.13; the exponential's argument in f32: |z| below 32 matters, 2^-23 each of it, and two roundings
    check(got, y / (1 + np.exp(-z)), mag[0] + 3, k, slope=1.2, rel=2.0**-18)


@gpu
def test_weight_as_the_right_operand_and_broadcast(device):
    weight, x, _, exact, mag = operands(device, (), 70, 320, 6)
    got = Tensor.from_data(x, None, device).matmul(weight, False, True).resolve().to(Device.CPU).storage
    check(got, exact[0], mag[0], 320)
    x3 = np.stack([x, x[::-1]])  # one weight for every element of a stack
    got = weight.gemm(Tensor.from_data(x3, None, device), None, False, True, True).resolve().to(Device.CPU).storage
    check(got, np.stack([exact[0], exact[0][::-1]]), np.stack([mag[0], mag[0][::-1]]), 320)
    # activations that are not contiguous along K
    got = weight.gemm(Tensor.from_data(np.ascontiguousarray(x.T), None, device), None, False, False, False).resolve().to(Device.CPU).storage
    check(got.T, exact[0], mag[0], 320)


@gpu
@pytest.mark.parametrize("n", [1, 3, 20, 100])
def test_infinities_and_nan_keep_to_their_rows(device, n):
    """An infinite activation times a positive, negative and zero weight is what the formula says; other rows are untouched."""
    m, k = 40, 2560
    codes, d = draw(m * k, 3)
    d[d == 0] = np.float16(0.01)
    d = np.abs(d)
    codes = codes.reshape(m, k)
    codes[:, 77] = np.array([0, 8, 15, 3] * 10)
    x = np.random.default_rng(1).standard_normal((n, k)).astype(np.float16)
    w = Tensor.from_quantized(segments(codes.reshape(-1), d), DType.Q4_0, (m, k), device)
    clean = w.gemm(Tensor.from_data(x, None, device), None, False, True, True).resolve().to(Device.CPU).storage
    x[n - 1, 77] = np.inf
    got = w.gemm(Tensor.from_data(x, None, device), None, False, True, True).resolve().to(Device.CPU).storage
    assert np.array_equal(got[: n - 1], clean[: n - 1])
    last = got[n - 1]
    assert (last[0::4] == -np.inf).all() and np.isnan(last[1::4]).all() and (last[2::4] == np.inf).all() and (last[3::4] == -np.inf).all()


@gpu
@pytest.mark.parametrize("n", [1, 20, 100])
def test_unaligned_activations_and_outputs(device, n):
    """Activations and outputs that start off 16 bytes go to another kernel, or the same, with the same results to the tolerance."""
    weight, x, _, exact, mag = operands(device, (), 65, 256, n)
    store = torch.zeros(2 * x.size + 64, dtype=torch.uint8, device="cuda:0")
    store[2 : 2 + 2 * x.size] = torch.from_numpy(x.view(np.uint8).reshape(-1)).to("cuda:0")
    out = torch.full((2 * 65 * n + 64,), 0xFF, dtype=torch.uint8, device="cuda:0")
    L, desc = _ffi.lib(), _ffi.make_desc(_ffi.RT_Q4_0, (65, 256), _ffi.RT_F16, (n, 256), False, True, True)
    st = L.rt_matmul_enqueue(device.ctx, ctypes.byref(desc), weight.data_ptr(), store.data_ptr() + 2, None, out.data_ptr() + 2, None)
    assert st == _ffi.RT_OK
    torch.cuda.synchronize()
    got = out[2 : 2 + 2 * 65 * n].cpu().numpy().view(np.float16).reshape(n, 65)
    check(got, exact[0], mag[0], 256)
    assert (out[:2] == 0xFF).all() and (out[2 + 2 * 65 * n :] == 0xFF).all()
    st = L.rt_matmul_enqueue(device.ctx, ctypes.byref(desc), weight.data_ptr().value + 2, store.data_ptr(), None, out.data_ptr(), None)
    assert st == _ffi.RT_ERR_UNSUPPORTED  # a weight off 16 bytes
