"""Products with Q4_0 weights on both sides of the lines that choose a kernel: rows and K that a tile or a unit of K ends in, the number of activation rows, a workspace
to share K in or none, plans, graphs and streams.  Layout, reference and tolerance are those of test_q4_0."""
import ctypes

import numpy as np
import pytest
import torch

from ratchet_amd import DType, Tensor, _ffi
from test_q4_0 import check, draw, operands, segments, values

gpu = pytest.mark.gpu


def call(device, weight, x, m, k, n, bias=None, how="enqueue", workspace=True):
    """[n, m] f16 of x [n, k] by the given entry point."""
    L = _ffi.lib()
    desc = _ffi.make_desc(_ffi.RT_Q4_0, (m, k), _ffi.RT_F16, (n, k), False, True, True, _ffi.RT_F16 if bias is not None else None, (m,) if bias is not None else None)
    need = ctypes.c_uint64()
    assert L.rt_matmul_workspace_bytes(device.ctx, ctypes.byref(desc), ctypes.byref(need)) == 0
    ws = torch.full((need.value + 64,), 0xFF, dtype=torch.uint8, device="cuda:0") if need.value and workspace else None
    out = torch.full((n * m + 8,), float("nan"), dtype=torch.float16, device="cuda:0")
    out[n * m :] = 7
    b = None if bias is None else bias.data_ptr()
    wp, wn = (ws.data_ptr(), need.value) if ws is not None else (None, 0)
    stream = torch.cuda.current_stream().cuda_stream
    if how == "plan":
        plan = ctypes.c_void_p()
        assert L.rt_matmul_plan_create(device.ctx, ctypes.byref(desc), _ffi.RT_ACT_NONE, ctypes.byref(plan)) == 0
        for _ in range(2):  # the second time the plan knows who took it
            out[: n * m] = float("nan")
            assert L.rt_matmul_plan_enqueue(plan, weight.data_ptr(), x.data_ptr(), b, out.data_ptr(), wp, wn, stream) == 0
        torch.cuda.synchronize()
        L.rt_matmul_plan_destroy(plan)
    else:
        assert L.rt_matmul_enqueue_ws(device.ctx, ctypes.byref(desc), weight.data_ptr(), x.data_ptr(), b, out.data_ptr(), _ffi.RT_ACT_NONE, wp, wn, stream) == 0
    assert (out[n * m :] == 7).all() and (ws is None or (ws[need.value :] == 0xFF).all())
    return out[: n * m].reshape(n, m), need.value


# weight rows, K: ends in a tile of 16, in eight outputs of a thread, in a unit of 512, 256, 128 of K; the generic kernel's K; rows below and from 160
LINES = [(15, 128), (24, 96), (161, 544), (168, 640), (320, 1024), (159, 256), (160, 256), (1025, 160), (2577, 1056), (640, 3840), (96, 5152)]
COUNTS = [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 63, 64, 65, 96, 97, 160, 257]


@gpu
@pytest.mark.parametrize("m,k", LINES)
def test_counts_of_activation_rows(device, m, k):
    for n in COUNTS:
        weight, x, bias, exact, mag = operands(device, (), m, k, n)
        xt, bt = torch.from_numpy(x).to("cuda:0"), torch.from_numpy(bias[0]).to("cuda:0")
        off = bias[0].astype(np.float64)
        first = None
        for how, ws in (("enqueue", True), ("plan", True), ("enqueue", False), ("plan", False)):
            got, need = call(device, weight, xt, m, k, n, bt, how, ws)
            check(got, exact[0] + off, mag[0] + np.abs(off), k)
            if how == "enqueue":
                first = got
            else:
                assert torch.equal(first.view(torch.int16), got.view(torch.int16)), (n, ws)  # a plan runs what a call runs


@gpu
@pytest.mark.parametrize("m,k,n", [(2560, 10240, 65), (2560, 10240, 160), (1280, 5120, 128), (4096, 4096, 160), (4097, 2560, 72), (512, 8192, 512)])
def test_shared_k_and_whole(device, m, k, n):
    """Shapes on both sides of the tiles' choice, with a workspace and without; the sums of shares are joined in a fixed order."""
    weight, x, bias, exact, mag = operands(device, (), m, k, n)
    xt = torch.from_numpy(x).to("cuda:0")
    for ws in (True, False):
        got, need = call(device, weight, xt, m, k, n, None, "enqueue", ws)
        again, _ = call(device, weight, xt, m, k, n, None, "plan", ws)
        check(got, exact[0], mag[0], k)
        assert torch.equal(got.view(torch.int16), again.view(torch.int16)), (ws, need)


@gpu
@pytest.mark.parametrize("n", [1, 7, 40, 200])
def test_products_captured_into_a_graph(device, n):
    """Two products, the second on the first's output, in a graph of another stream, replayed over changing activations beside the eager calls."""
    m, k = 768, 1536
    (w1, x, _, _, _), (w2, _, _, _, _) = operands(device, (), m, k, n), operands(device, (), k, m, n)
    xt = torch.from_numpy(x).to("cuda:0") * 0.05
    L = _ffi.lib()
    d1, d2 = (_ffi.make_desc(_ffi.RT_Q4_0, s, _ffi.RT_F16, (n, s[1]), False, True, True) for s in ((m, k), (k, m)))
    need = ctypes.c_uint64()
    size = 64
    for d in (d1, d2):
        assert L.rt_matmul_workspace_bytes(device.ctx, ctypes.byref(d), ctypes.byref(need)) == 0
        size = max(size, need.value)
    y = [torch.empty((n, m), dtype=torch.float16, device="cuda:0") for _ in range(2)]
    z = [torch.empty((n, k), dtype=torch.float16, device="cuda:0") for _ in range(2)]
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda:0") for _ in range(2)]

    def both(i, stream):
        for d, w, a, o in ((d1, w1, xt, y[i]), (d2, w2, y[i], z[i])):
            assert L.rt_matmul_enqueue_ws(device.ctx, ctypes.byref(d), w.data_ptr(), a.data_ptr(), None, o.data_ptr(), 0, ws[i].data_ptr(), size, stream) == 0

    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        both(0, torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        xt.mul_(-0.8)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        both(1, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.isfinite(z[0]).all() and torch.equal(z[0].view(torch.int16), z[1].view(torch.int16)), i


@gpu
@pytest.mark.parametrize("m,k,n", [(40, 288, 4097), (163, 128, 1500), (33, 96, 700)])
def test_many_activation_rows_against_few_weights(device, m, k, n):
    weight, x, bias, exact, mag = operands(device, (), m, k, n)
    got, _ = call(device, weight, torch.from_numpy(x).to("cuda:0"), m, k, n)
    check(got, exact[0], mag[0], k)


@gpu
@pytest.mark.parametrize("m,k,n", [(2560, 10240, 96), (512, 2048, 4), (640, 2048, 512)])
def test_the_form_without_a_workspace_argument(device, m, k, n):
    """rt_matmul_enqueue_static: Q4_0 weights run there as they do without a workspace."""
    weight, x, _, exact, mag = operands(device, (), m, k, n)
    xt = torch.from_numpy(x).to("cuda:0")
    plain, _ = call(device, weight, xt, m, k, n, workspace=False)
    desc = _ffi.make_desc(_ffi.RT_Q4_0, (m, k), _ffi.RT_F16, (n, k), False, True, True)
    out = torch.full((n, m), float("nan"), dtype=torch.float16, device="cuda:0")
    assert _ffi.lib().rt_matmul_enqueue_static(device.ctx, ctypes.byref(desc), weight.data_ptr(), xt.data_ptr(), None, out.data_ptr(), _ffi.RT_ACT_NONE,
                                               torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16))
    check(out, exact[0], mag[0], k)


@gpu
@pytest.mark.parametrize("n", [1, 2, 3, 9, 40, 200])
def test_subnormal_activations(device, n):
    """Activations below f16's normal range count like any others; weights of the largest scales keep the products in it."""
    rng = np.random.default_rng(n)
    m, k = 170, 2048
    codes, d = draw(m * k, n)
    d = np.full_like(d, 8000)
    x = (rng.integers(-1023, 1024, (n, k)) * 2.0**-24).astype(np.float16)
    w = values(codes, d).reshape(m, k)
    weight = Tensor.from_quantized(segments(codes, d), DType.Q4_0, (m, k), device)
    got, _ = call(device, weight, torch.from_numpy(x).to("cuda:0"), m, k, n)
    xd = x.astype(np.float64)
    check(got, xd @ w.T, np.abs(xd) @ np.abs(w).T, k)


# K that lanes of a row share evenly, that leaves lanes without a block, one block; K that two, three, four wavefronts share; rows that end in a group of four and many passes
@gpu
@pytest.mark.parametrize("k", [32, 64, 512, 544, 2528, 2560, 2592, 5120, 5152, 7680, 10240, 10272])
@pytest.mark.parametrize("m", [1, 7, 2050, 9001])
def test_one_and_two_vectors(device, m, k):
    for n in (1, 2):
        weight, x, bias, exact, mag = operands(device, (), m, k, n)
        xt, bt = torch.from_numpy(x).to("cuda:0"), torch.from_numpy(bias[0]).to("cuda:0")
        off = bias[0].astype(np.float64)
        got, _ = call(device, weight, xt, m, k, n, bt)
        check(got, exact[0] + off, mag[0] + np.abs(off), k)
        if m == 7:
            x[n - 1, k - 1] = np.inf  # the last value of the last vector: others are untouched, and no lane without a block sees it
            clean = got
            got, _ = call(device, weight, torch.from_numpy(x).to("cuda:0"), m, k, n, bt)
            assert torch.equal(got[: n - 1], clean[: n - 1]) and not torch.isfinite(got[n - 1]).any()
