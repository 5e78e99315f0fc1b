"""The key/value cache held in pages: the write (bit for bit the rows it is given, everything else untouched) and the attention over it against the
operator in 64 bits (ragged_cases has the tolerance)."""
import ctypes
import math

import pytest
import torch

from ragged_cases import Paged, attend_paged, cache_desc, close, paged_desc, reference, starts_of, stream, write_paged
from ratchet_amd import _ffi

gpu = pytest.mark.gpu


# ---- the write ------------------------------------------------------------------------------------------------------------------


def written(pool, table, lens, n, src, page_size):
    """The pool after the write, row by row."""
    pool, at = pool.clone(), 0
    for b, rows in enumerate(n):
        for i in range(rows):
            p = lens[b] - rows + i
            page = int(table[b, p // page_size]) if 0 <= p < table.shape[1] * page_size else -1
            if 0 <= page < pool.shape[0]:
                pool[page, :, p % page_size] = src[at + i].half()
        at += rows
    return pool


def write_case(device, seed, n, before, kv, d, page_size, dtype=torch.float16, one=False, table_stride=0):
    gen = torch.Generator().manual_seed(seed)
    lens = [x + y for x, y in zip(n, before)]
    pages = sum((x + page_size - 1) // page_size for x in lens) + 2
    width = max(1, max((x + page_size - 1) // page_size for x in lens))
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(n), width + table_stride), -1, dtype=torch.int32)
    for i, x in enumerate(lens):
        for j in range((x + page_size - 1) // page_size):
            table[i, j] = order.pop()
    rows = sum(n) + 2
    k, v = (torch.randn((rows, kv, d), generator=gen).to(dtype) for _ in range(2))
    pools = [torch.randn((pages, kv, page_size, d), generator=gen).half() for _ in range(2)]
    gpu_pools = [x.cuda() for x in pools]
    cache = cache_desc(len(n), kv, d, pages, page_size, width, width + table_stride)
    write_paged(device, cache, gpu_pools[0], k.cuda(), None if one else gpu_pools[1], None if one else v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                starts_of(n).cuda(), rows)
    assert torch.equal(gpu_pools[0].cpu(), written(pools[0], table[:, :width], lens, n, k, page_size))
    assert torch.equal(gpu_pools[1].cpu(), pools[1] if one else written(pools[1], table[:, :width], lens, n, v, page_size))


@gpu
@pytest.mark.parametrize("n,before", [([1], [0]), ([1, 1, 1], [0, 15, 16]), ([0, 5, 0, 40, 0], [3, 14, 0, 100, 0]), ([1] * 130, list(range(130))), ([0] * 70 + [3], [0] * 71), ([257], [31])],
                         ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_write(device, n, before, dtype):
    write_case(device, len(n), n, before, 2, 80, 16, dtype)


@gpu
@pytest.mark.parametrize("kv,d,page_size", [(1, 8, 16), (8, 128, 64), (3, 72, 1024), (40, 64, 32)])
def test_write_layouts(device, kv, d, page_size):
    write_case(device, kv, [3, 17, 1], [60, 0, 15], kv, d, page_size, table_stride=5)
    write_case(device, kv, [3, 17, 1], [60, 0, 15], kv, d, page_size, one=True)


@gpu
def test_write_of_parts_of_a_projection_and_without_starts(device):
    b, n, kv, d, ps = 3, 4, 2, 64, 16
    gen = torch.Generator().manual_seed(2)
    for dtype in (torch.float16, torch.float32):
        qkv = torch.randn((b * n, 5 * kv * d), generator=gen).to(dtype)
        k, v = qkv[:, 3 * kv * d:4 * kv * d], qkv[:, 4 * kv * d:]
        table = torch.tensor([[4, 1], [0, 2], [3, 5]], dtype=torch.int32)
        lens = [14, 20, 4]
        pools = [torch.zeros((6, kv, ps, d), dtype=torch.float16) for _ in range(2)]
        on = [x.cuda() for x in pools]
        x = qkv.cuda()
        write_paged(device, cache_desc(b, kv, d, 6, ps, 2), on[0], x[:, 3 * kv * d:], on[1], x[:, 4 * kv * d:], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), None, b * n,
                    [5 * kv * d, d])
        for got, want, src in zip(on, pools, (k, v)):
            assert torch.equal(got.cpu(), written(want, table, lens, [n] * b, src.reshape(b * n, kv, d), ps))


@gpu
def test_places_outside_are_not_written(device):
    """Positions below 0 and past the table, entries that are no page, starts that point outside or descend."""
    kv, d, ps = 1, 64, 16
    table = torch.tensor([[0, -1, 7], [1, 99, -2147483648], [2, 3, 2147483647]], dtype=torch.int32)
    src = torch.randn((60, kv, d), generator=torch.Generator().manual_seed(0)).half()
    for n, lens in (([20, 20, 20], [10, 30, 50]), ([20, 20, 20], [60, 0, -7]), ([20, 20, 20], [2**31 - 1, -2**31, 2**31 - 5])):
        pool = torch.full((4, kv, ps, d), 5.0, dtype=torch.float16)
        on = pool.cuda()
        write_paged(device, cache_desc(3, kv, d, 4, ps, 3), on, src.cuda(), None, None, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts_of(n).cuda(), 60)
        assert torch.equal(on.cpu(), written(pool, table, lens, n, src, ps)), lens
    for starts in ([50, 10, 70, 20], [-2**31, 2**31 - 1, -1, 5], [-5, 10, 20, 30]):
        on = torch.zeros((4, kv, ps, d), dtype=torch.float16, device="cuda")
        write_paged(device, cache_desc(3, kv, d, 4, ps, 3), on, src.cuda(), None, None, table.cuda(), torch.tensor([16, 16, 32], dtype=torch.int32).cuda(),
                    torch.tensor(starts, dtype=torch.int32).cuda(), 60)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(on).all())


# ---- the attention ----------------------------------------------------------------------------------------------------------------


def attend(device, seed, n, lens, heads, kv, d, page_size, causal=True, max_rows=None, max_keys=None, scale=None, workspace=True, sharp=1.0, hidden=None):
    c = Paged(seed, lens, kv, d, page_size, max_keys, sharp)
    if hidden:   # pages taken out of the table: nobody sees their keys
        for b, j in hidden:
            c.table[b, j] = (-1, c.cache.pages, 2**31 - 1, -2**31)[(b + j) % 4]
    scale = 1 / math.sqrt(d) if scale is None else scale
    rows = sum(n) + 2
    q = torch.randn((rows, heads, d), generator=torch.Generator().manual_seed(seed + 1)).half()
    gone = [[p for j in range(c.width) if (b, j) in hidden for p in range(j * page_size, min(lens[b], (j + 1) * page_size))] for b in range(len(n))] if hidden else None
    want, tol = reference(q[: sum(n)], c.k, c.v, n, lens, scale, causal, gone)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    desc = paged_desc(c.cache, heads, rows, max(n) if max_rows is None else max_rows, c.width * page_size if max_keys is None else max_keys, causal, scale)
    k_pool, v_pool, table, on_lens = c.on_gpu()
    attend_paged(device, desc, q.cuda(), k_pool, v_pool, table, on_lens, starts_of(n).cuda(), out, workspace)
    close(out[: sum(n)], want, tol, (n, lens, heads, kv, d, page_size, causal))
    assert bool((out[sum(n):] == 7.0).all())
    return out


@gpu
@pytest.mark.parametrize("d", [8, 24, 40, 64, 72, 80, 96, 112, 120, 128])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_head_sizes(device, d, rows):
    attend(device, d, [rows, rows, rows], [rows + 130, rows, rows + 31], 4, 2, d, 16)


@gpu
@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 1024, 65536])
@pytest.mark.parametrize("rows", [1, 40])
def test_page_sizes(device, page_size, rows):
    attend(device, page_size, [rows, rows], [rows + 300, rows + 17], 2, 2, 64, page_size)
    attend(device, page_size, [rows], [rows + 1100], 4, 1, 128, page_size)


@gpu
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [31, 32, 33, 63, 64, 65], [127, 128, 129], [0, 5, 0], [1000, 3, 2047, 2048, 2049], [7] * 90, [40] * 300], ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2), (16, 1)])
def test_one_row(device, lens, heads, kv):
    attend(device, len(lens), [1] * len(lens), lens, heads, kv, 128, 16)


@gpu
@pytest.mark.parametrize("rows", [2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
def test_a_few_rows(device, rows, heads, kv):
    """Drafted tokens: each sees the ones before it."""
    attend(device, rows, [rows, rows, max(1, rows - 1), 0, 1], [rows + 200, rows, 1000, 50, 77], heads, kv, 96, 32, max_rows=rows)


@gpu
@pytest.mark.parametrize("rows", [1, 4, 50])
def test_without_the_causal_flag(device, rows):
    attend(device, rows, [rows] * 3, [100, 9, 700], 4, 2, 64, 16, causal=False)


@gpu
@pytest.mark.parametrize("rows", [1, 3, 90])
def test_more_rows_than_keys(device, rows):
    """Rows that see no key are NaN; a sequence with none."""
    attend(device, rows, [rows, rows, rows], [0, max(0, rows - 2), rows + 40], 2, 2, 80, 16)


@gpu
@pytest.mark.parametrize("d", [8, 24, 40, 64, 72, 88, 104, 128])
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("lens", [[129, 255, 256, 257, 0, 1, 500, 512], [160, 288, 511] * 40], ids=["few", "many"])
def test_a_few_steps(device, rows, d, lens):
    """Heads of keys of two to four steps, fewer and more of them than there are compute units."""
    attend(device, rows + d, [min(rows, x) for x in lens], lens, 12, 3, d, 16)
    attend(device, rows + d, [min(rows, x) for x in lens], lens, 12, 3, d, 16, causal=False, hidden={(0, 3), (2, 15), (3, 2)})


@gpu
@pytest.mark.parametrize("rows,lens", [(1, [9000]), (1, [20000, 5, 3000]), (6, [9001]), (40, [9000, 100]), (200, [3000])])
@pytest.mark.parametrize("workspace", [True, False])
def test_long_sequences(device, rows, lens, workspace):
    attend(device, rows, [min(rows, x) for x in lens], lens, 4, 2, 128, 16, workspace=workspace)


@gpu
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_bounds_far_above_the_lengths(device, rows):
    """max_rows and max_keys are bounds: calls captured for longer sequences than there are."""
    attend(device, rows, [rows, rows], [rows + 20, rows + 333], 4, 2, 64, 16, max_rows=rows, max_keys=16384)
    attend(device, rows, [rows, rows], [rows + 20, rows + 333], 4, 2, 64, 16, max_rows=500, max_keys=16384)


@gpu
@pytest.mark.parametrize("batch,kv,d,most,rows", [(150, 2, 64, 2000, 2), (300, 1, 40, 1500, 1), (300, 8, 16, 700, 1), (65, 3, 96, 900, 5), (64, 1, 128, 3000, 8), (100, 1, 64, 2500, 2), (130, 1, 96, 3000, 1), (70, 2, 128, 2500, 3)])
def test_many_sequences_share_workgroups(device, batch, kv, d, most, rows):
    """Parts of one workgroup end and begin within sequences of any length, empty ones and ones without rows among them; from 2048 heads of keys on each has a workgroup."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, most, (batch,), generator=gen).tolist()
    n = torch.randint(0, rows + 1, (batch,), generator=gen).tolist()
    n[0], lens[0], n[1], n[-1] = rows, most, 0, rows
    attend(device, batch, n, lens, 2 * kv, kv, d, 16, max_rows=rows)


@gpu
def test_more_rows_than_promised(device):
    """Sequences are cut to max_rows rows: what lies past them is left as it was, and the others are right."""
    c = Paged(3, [700, 90], 2, 64, 16)
    q = torch.randn((12, 4, 64), generator=torch.Generator().manual_seed(2)).half()
    k_pool, v_pool, table, lens = c.on_gpu()
    want, tol = reference(q[9:], [c.k[1]], [c.v[1]], [3], [90], 0.125, True)
    for rows in (3, 40):     # on both kernels
        x = torch.cat([q[:9].repeat_interleave(rows // 3, 0), q[9:].repeat_interleave(1, 0)])
        first = 9 * (rows // 3)
        out = torch.full(x.shape, 7.0, dtype=torch.float16, device="cuda")
        starts = torch.tensor([0, first, first + 3], dtype=torch.int32).cuda()
        attend_paged(device, paged_desc(c.cache, 4, first + 3, rows, c.width * 16, True, 0.125), x.cuda(), k_pool, v_pool, table, lens, starts, out)
        assert bool((out[rows:first] == 7.0).all()) and bool(torch.isfinite(out[:rows]).all())
        close(out[first:], want, tol, rows)


@gpu
@pytest.mark.parametrize("rows", [1, 9, 60])
def test_pages_that_are_not_there(device, rows):
    """Entries outside the pool, at the beginning (what has left a window), in the middle, at the end, and all of a sequence's."""
    hidden = {(0, 0), (0, 1), (0, 7), (1, 3), (2, 12)} | {(3, j) for j in range(5)}
    attend(device, rows, [rows] * 4, [rows + 200, rows + 100, 203, min(80, rows + 70)], 4, 2, 64, 16, hidden=hidden)
    attend(device, rows, [rows] * 2, [rows + 900, rows + 300], 2, 1, 128, 64, hidden={(0, 0), (0, 1), (0, 2), (1, 1)})


@gpu
@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0, 1e-20])
def test_scales(device, rows, scale):
    attend(device, 3, [rows] * 2, [rows + 400, rows], 4, 2, 64, 16, scale=scale)


@gpu
@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("sharp", [40.0, 3000.0])
def test_large_scores(device, rows, sharp):
    attend(device, 4, [rows] * 2, [rows + 1400, rows + 7], 4, 2, 128, 16, sharp=sharp)


@gpu
@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("size", [1.0, 60000.0])
def test_equal_keys_weigh_the_same(device, rows, size):
    """Keys alike, scores up to 2^39, shares of a long sequence: the mean of the values."""
    n, d, ps = 5000, 128, 64
    c = Paged(1, [n], 1, d, ps)
    c.k = [torch.full((n, 1, d), size, dtype=torch.float16)]
    c.fill()
    k_pool, v_pool, table, lens = c.on_gpu()
    q = torch.full((rows, 2, d), size, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    attend_paged(device, paged_desc(c.cache, 2, rows, rows, n, True, 1.0), q, k_pool, v_pool, table, lens, None, out)
    v = c.v[0].double()
    for i in range(rows):
        seen = n - rows + i + 1
        mean, size_of = v[:seen, 0].mean(0), v[:seen, 0].abs().mean(0)
        close(out[i], mean.expand(2, d), (n * 2.0**-24 * 2 * size_of + 2.0**-11 * mean.abs() + 2.0**-25).expand(2, d), (rows, size, i))


@gpu
@pytest.mark.parametrize("rows", [1, 6, 60])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_keys_have_no_effect(device, rows, d):
    """NaN and infinities behind a sequence's keys (the rest of its pages is NaN anyway) and in keys that some rows do not see."""
    n, lens = [rows, rows], [rows + 150, rows + 40]
    c = Paged(5, lens, 2, d, 16)
    q = torch.randn((2 * rows, 4, d), generator=torch.Generator().manual_seed(6)).half()
    want, tol = reference(q, c.k, c.v, n, lens, 0.1, True)
    at = rows // 2   # the row of the first sequence from which on a NaN is seen, and in the second an infinity of each sign
    p0, p1 = lens[0] - rows + at, lens[1] - rows + at
    c.k[0][p0], c.v[0][p0] = float("nan"), float("nan")
    c.v[1][p1, 0, 3], c.v[1][p1, 1, 5] = float("inf"), float("-inf")
    c.fill()
    k_pool, v_pool, table, on_lens = c.on_gpu()
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    attend_paged(device, paged_desc(c.cache, 4, 2 * rows, rows, c.width * 16, True, 0.1), q.cuda(), k_pool, v_pool, table, on_lens, starts_of(n).cuda(), out)
    got, odd = out.double().cpu(), torch.zeros(q.shape, dtype=torch.bool)
    odd[at:rows] = True
    odd[rows + at:, :2, 3] = True
    odd[rows + at:, 2:, 5] = True
    assert not bool(torch.isfinite(got[odd]).any())
    close(torch.where(odd, want, got), want, tol)


@gpu
@pytest.mark.parametrize("rows", [1, 7, 50])
def test_pages_that_sequences_share(device, rows):
    """A prefix that two sequences have in common, and a page twice in one sequence: each sees what its own row of the table names."""
    c = Paged(11, [200, 150], 2, 64, 16)
    c.table[1, :5] = c.table[0, :5]
    c.table[1, 7] = c.table[1, 6]
    pages = [c.table[i, : (n + 15) // 16].long() for i, n in enumerate(c.lens)]
    k, v = ([pool[p].transpose(1, 2).reshape(-1, 2, 64)[:n] for p, n in zip(pages, c.lens)] for pool in (c.k_pool, c.v_pool))
    q = torch.randn((2 * rows, 4, 64), generator=torch.Generator().manual_seed(1)).half()
    want, tol = reference(q, k, v, [rows, rows], c.lens, 0.125, True)
    k_pool, v_pool, table, lens = c.on_gpu()
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    attend_paged(device, paged_desc(c.cache, 4, 2 * rows, rows, c.width * 16, True, 0.125), q.cuda(), k_pool, v_pool, table, lens, None, out)
    close(out, want, tol)


@gpu
def test_no_pages_and_no_table(device):
    q = torch.randn((3, 2, 64)).half().cuda()
    for pages, width in ((0, 4), (4, 0)):
        out = torch.zeros_like(q)
        pool = torch.zeros((max(pages, 1), 1, 16, 64), dtype=torch.float16, device="cuda")
        table, lens = torch.zeros((3, max(width, 1)), dtype=torch.int32, device="cuda"), torch.full((3,), 9, dtype=torch.int32, device="cuda")
        desc = paged_desc(cache_desc(3, 1, 64, pages, 16, width), 2, 3, 1, 64 if width else 0, True, 0.1)
        attend_paged(device, desc, q, pool, pool, table, lens, None, out)
        assert bool(torch.isnan(out).all())


@gpu
def test_lens_outside_their_bounds(device):
    """lens below 0 and past max_keys are taken as those."""
    c = Paged(7, [160], 1, 64, 16)
    q = torch.randn((1, 1, 64), generator=torch.Generator().manual_seed(1)).half()
    k_pool, v_pool, table, _ = c.on_gpu()
    want, tol = reference(q, [x[:100] for x in c.k], [x[:100] for x in c.v], [1], [100], 0.1, True)
    for n in (101, 2**31 - 1, -1, -2**31):
        out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
        attend_paged(device, paged_desc(c.cache, 1, 1, 1, 100, True, 0.1), q.cuda(), k_pool, v_pool, table, torch.tensor([n], dtype=torch.int32).cuda(), None, out)
        if n > 0:
            close(out, want, tol)
        else:
            assert bool(torch.isnan(out).all())


@gpu
def test_pools_past_4_gib(device):
    """Pages whose bytes lie past 2^32: the write and the attention of one row, a few, and many."""
    kv, d, ps = 8, 128, 256
    pages = 2**33 // (kv * d * ps * 2) + 8          # 8 GiB a pool
    k_pool, v_pool = (torch.zeros((pages, kv, ps, d), dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 1, pages - 2, pages // 2 + 1]], dtype=torch.int32)
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn((900, kv, d), generator=gen).half() for _ in range(2))
    cache, lens = cache_desc(1, kv, d, pages, ps, 4), torch.tensor([900], dtype=torch.int32).cuda()
    write_paged(device, cache, k_pool, k.cuda(), v_pool, v.cuda(), table.cuda(), lens, starts_of([900]).cuda(), 900)
    for pool, x in ((k_pool, k), (v_pool, v)):
        rows = pool[table[0].long().cuda()].transpose(1, 2).reshape(-1, kv, d)[:900].cpu()
        assert torch.equal(rows, x)
    for rows in (1, 7, 300):
        q = torch.randn((rows, kv, d), generator=gen).half()
        want, tol = reference(q, [k], [v], [rows], [900], 0.09, True)
        out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
        attend_paged(device, paged_desc(cache, kv, rows, rows, 900, True, 0.09), q.cuda(), k_pool, v_pool, table.cuda(), lens, None, out)
        close(out, want, tol, rows)


@gpu
@pytest.mark.parametrize("rows", [1, 3, 100])
def test_a_serving_loop(device, rows):
    """Write and attend as they are used: a prompt each, then steps, with a captured graph of both whose lengths and tables change between replays."""
    b, heads, kv, d, ps, cap = 3, 4, 2, 64, 16, 40
    gen = torch.Generator().manual_seed(8)
    prompts = [5, 33, 17]
    pages, width = 3 * cap, cap
    table = torch.randperm(pages, generator=gen).view(3, cap).to(torch.int32)
    k_pool, v_pool = (torch.full((pages, kv, ps, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    cache = cache_desc(b, kv, d, pages, ps, width)
    on_table, lens = table.cuda(), torch.tensor(prompts, dtype=torch.int32).cuda()
    k, v = ([torch.randn((x, kv, d), generator=gen).half() for x in prompts] for _ in range(2))
    write_paged(device, cache, k_pool, torch.cat(k).cuda(), v_pool, torch.cat(v).cuda(), on_table, lens, starts_of(prompts).cuda(), sum(prompts))
    new_k, new_v = (torch.zeros((b * rows, kv, d), dtype=torch.float16, device="cuda") for _ in range(2))
    q, out = (torch.zeros((b * rows, heads, d), dtype=torch.float16, device="cuda") for _ in range(2))
    desc = paged_desc(cache, heads, b * rows, rows, cap * ps, True, 0.125)
    need = ctypes.c_uint64()
    assert _ffi.lib().rt_attention_paged_workspace_bytes(desc, need) == _ffi.RT_OK
    ws = torch.full((max(need.value, 1),), 0xFF, dtype=torch.uint8, device="cuda")

    def once():
        write_paged(device, cache, k_pool, new_k, v_pool, new_v, on_table, lens, None, b * rows)
        attend_paged(device, desc, q, k_pool, v_pool, on_table, lens, None, out, ws)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once()
    for step in range(4):
        x, y, z = (torch.randn(s, generator=gen).half() for s in ((b * rows, kv, d), (b * rows, kv, d), (b * rows, heads, d)))
        new_k.copy_(x), new_v.copy_(y), q.copy_(z)
        k, v = ([torch.cat([old, new]) for old, new in zip(a, new.split(rows))] for a, new in ((k, x), (v, y)))
        sizes = [len(a) for a in k]
        lens.copy_(torch.tensor(sizes, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay() if step % 2 == 0 else once()
        want, tol = reference(z, k, v, [rows] * b, sizes, 0.125, True)
        close(out, want, tol, step)
    first = out.clone()
    for _ in range(3):   # the same inputs again: the same bits
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


@gpu
def test_two_streams_and_workspaces(device):
    """Two calls at once on streams of their own with workspaces of their own."""
    cases = []
    for seed, lens in ((1, [9000, 50]), (2, [300, 12000])):
        c = Paged(seed, lens, 2, 64, 16)
        q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(seed)).half()
        cases.append((c, q, reference(q, c.k, c.v, [1, 1], lens, 0.125, True), c.on_gpu(), paged_desc(c.cache, 4, 2, 1, max(lens), True, 0.125)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    torch.cuda.synchronize()
    for _ in range(3):
        outs = []
        for s, (c, q, _, t, desc) in zip(streams, cases):
            with torch.cuda.stream(s):
                outs.append(attend_paged(device, desc, q.cuda(), *t[:2], t[2], t[3], None, torch.empty(q.shape, dtype=torch.float16, device="cuda")))
        torch.cuda.synchronize()
        for out, (c, q, (want, tol), t, desc) in zip(outs, cases):
            close(out, want, tol)


# ---- what is refused -------------------------------------------------------------------------------------------------------------


def fine():
    return paged_desc(cache_desc(2, 2, 64, 10, 16, 4), 8, 10, 8, 64, True, 0.125)


@pytest.mark.parametrize("field,value,status", [
    ("batch", -1, _ffi.RT_ERR_INVALID_SHAPE), ("kv_heads", -1, _ffi.RT_ERR_INVALID_SHAPE), ("kv_heads", 3, _ffi.RT_ERR_INVALID_SHAPE), ("kv_heads", 0, _ffi.RT_ERR_INVALID_SHAPE),
    ("head_dim", 0, _ffi.RT_ERR_INVALID_SHAPE), ("head_dim", 20, _ffi.RT_ERR_INVALID_SHAPE), ("head_dim", 136, _ffi.RT_ERR_INVALID_SHAPE), ("pages", -1, _ffi.RT_ERR_INVALID_SHAPE),
    ("page_size", 0, _ffi.RT_ERR_INVALID_SHAPE), ("page_size", 8, _ffi.RT_ERR_INVALID_SHAPE), ("page_size", 48, _ffi.RT_ERR_INVALID_SHAPE), ("page_size", 131072, _ffi.RT_ERR_INVALID_SHAPE),
    ("table_width", -1, _ffi.RT_ERR_INVALID_SHAPE), ("table_width", 3, _ffi.RT_ERR_INVALID_SHAPE), ("table_stride", 3, _ffi.RT_ERR_INVALID_SHAPE), ("table_stride", -1, _ffi.RT_ERR_INVALID_SHAPE),
    ("batch", 65536, _ffi.RT_ERR_UNSUPPORTED), ("table_stride", 1 << 40, _ffi.RT_ERR_UNSUPPORTED),
])
def test_refused_caches(field, value, status):
    L, d, need = _ffi.lib(), fine(), ctypes.c_uint64()
    assert L.rt_attention_paged_validate(d) == _ffi.RT_OK
    setattr(d.cache, field, value)
    assert L.rt_attention_paged_validate(d) == status
    assert L.rt_attention_paged_workspace_bytes(d, need) == status


@pytest.mark.parametrize("field,value,status", [
    ("heads", -8, _ffi.RT_ERR_INVALID_SHAPE), ("heads", 7, _ffi.RT_ERR_INVALID_SHAPE), ("rows", -1, _ffi.RT_ERR_INVALID_SHAPE), ("max_rows", -1, _ffi.RT_ERR_INVALID_SHAPE),
    ("max_keys", -1, _ffi.RT_ERR_INVALID_SHAPE), ("max_keys", 65, _ffi.RT_ERR_INVALID_SHAPE), ("causal", 2, _ffi.RT_ERR_INVALID_ARG), ("scale", float("nan"), _ffi.RT_ERR_INVALID_ARG),
    ("scale", float("-inf"), _ffi.RT_ERR_INVALID_ARG), ("rows", (1 << 25) + 1, _ffi.RT_ERR_UNSUPPORTED), ("heads", 1 << 30, _ffi.RT_ERR_UNSUPPORTED),
])
def test_refused_attention(field, value, status):
    L, d, need = _ffi.lib(), fine(), ctypes.c_uint64()
    setattr(d, field, value)
    assert L.rt_attention_paged_validate(d) == status
    assert L.rt_attention_paged_workspace_bytes(d, need) == status


@pytest.mark.parametrize("name", ["q_strides", "o_strides"])
def test_refused_strides(name):
    for i in range(2):
        for value, status in ((-8, _ffi.RT_ERR_INVALID_SHAPE), (12, _ffi.RT_OK if name == "o_strides" else _ffi.RT_ERR_UNSUPPORTED), (1 << 40, _ffi.RT_ERR_UNSUPPORTED)):
            d = fine()
            getattr(d, name)[i] = value
            assert _ffi.lib().rt_attention_paged_validate(d) == status, (i, value)


def test_null_arguments():
    L, need = _ffi.lib(), ctypes.c_uint64()
    assert L.rt_attention_paged_validate(None) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_paged_workspace_bytes(None, need) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_paged_workspace_bytes(fine(), None) == _ffi.RT_ERR_INVALID_ARG
    assert L.rt_attention_paged_enqueue(None, fine(), None, None, None, None, None, None, None, None, 0, None) == _ffi.RT_ERR_INVALID_ARG
    s = (ctypes.c_int64 * 2)(64, 64)
    assert L.rt_cache_write_paged_enqueue(None, cache_desc(1, 1, 64, 1, 16, 1), _ffi.RT_F16, None, None, None, None, s, None, None, None, 1, None) == _ffi.RT_ERR_INVALID_ARG


@gpu
def test_refused_calls(device):
    L = _ffi.lib()
    z, s = torch.zeros(10 * 8 * 64 + 8, dtype=torch.float16, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    p, i = z.data_ptr(), s.data_ptr()
    good = [device.ctx, fine(), p, p, p, i, i, i, p, None, 0, None]
    for at, value, status in ((2, None, 1), (3, None, 1), (4, None, 1), (5, None, 1), (6, None, 1), (8, None, 1), (2, p + 2, 1), (3, p + 8, 1), (4, p + 8, 1), (5, i + 2, 1), (6, i + 1, 1),
                              (7, i + 2, 1), (8, p + 1, 1), (7, None, 2)):
        args = list(good)
        args[at] = value
        assert L.rt_attention_paged_enqueue(*args) == status, at
    strides = (ctypes.c_int64 * 2)(128, 64)
    good = [device.ctx, cache_desc(2, 2, 64, 10, 16, 4), _ffi.RT_F16, p, p, p, p, strides, i, i, i, 10, None]
    for at, value, status in ((1, None, 1), (2, _ffi.RT_Q8_0H, 3), (3, None, 1), (4, None, 1), (5, None, 1), (6, None, 1), (7, None, 1), (8, None, 1), (9, None, 1), (3, p + 8, 1), (4, p + 2, 1),
                              (5, p + 8, 1), (6, p + 2, 1), (7, (ctypes.c_int64 * 2)(-8, 64), 4), (7, (ctypes.c_int64 * 2)(12, 64), 4), (7, (ctypes.c_int64 * 2)(128, 1 << 40), 4),
                              (8, i + 1, 1), (9, i + 2, 1), (10, i + 2, 1), (11, -1, 2), (11, (1 << 25) + 1, 4), (1, cache_desc(2, 2, 60, 10, 16, 4), 2), (1, cache_desc(2, 2, 64, 10, 24, 4), 2)):
        args = list(good)
        args[at] = value
        assert L.rt_cache_write_paged_enqueue(*args) == status, (at, value)
    args = list(good)
    args[10], args[11] = None, 9      # without starts: rows / batch each
    assert L.rt_cache_write_paged_enqueue(*args) == _ffi.RT_ERR_INVALID_SHAPE
    for cache, rows in ((cache_desc(0, 2, 64, 10, 16, 4), 0), (cache_desc(2, 2, 64, 0, 16, 4), 10), (cache_desc(2, 2, 64, 10, 16, 0), 10), (cache_desc(2, 2, 64, 10, 16, 4), 0)):
        assert L.rt_cache_write_paged_enqueue(device.ctx, cache, _ffi.RT_F16, None, None, None, None, strides, None, None, None, rows, None) == _ffi.RT_OK   # nothing to do
    torch.cuda.synchronize()
    assert not bool(z.any())
