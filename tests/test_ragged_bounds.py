"""Sequences that are longer than a call's bounds, or reach past its tensors: the rows and keys that are left out are left out, and the rows that are kept see what they would
see without the bound (against the operator in 64 bits on the whole sequences; ragged_cases has the tolerance)."""
import pytest
import torch

from ragged_cases import Paged, attend_packed, attend_paged, close, packed_desc, paged_desc, reference, starts_of

gpu = pytest.mark.gpu


def kept_rows(n, max_rows, rows):
    """Packed rows that a call computes, of sequences one behind another in a tensor of so many rows."""
    at, kept = 0, []
    for x in n:
        kept += [r for r in range(at, at + x) if r < rows and r - at < max_rows]
        at += x
    return torch.tensor(kept, dtype=torch.long)


def compare(out, want, tol, kept, what):
    close(out[kept.cuda()], want[kept], tol[kept], what)
    left = torch.ones(out.shape[0], dtype=torch.bool)
    left[kept] = False
    assert bool((out[left.cuda()] == 7.0).all()), what


# n: the sequences' rows; max_rows and max_keys below them; rows: of the tensor, fewer than the sequences' in some
PAGED = [
    ([100, 3], [100, 50], 60, 112, None), ([9, 2], [700, 90], 3, 704, None), ([9, 2], [9, 90], 3, 96, None), ([20, 31, 5], [20, 2000, 700], 7, 2000, None),
    ([400, 129], [3000, 129], 130, 3008, None), ([3, 6], [40, 90], 6, 96, 6), ([40, 60], [90, 60], 60, 96, 70), ([200, 300], [200, 900], 300, 912, 450),
    ([5, 6], [90, 40], 6, 64, None), ([70, 80], [200, 90], 80, 112, None), ([5, 1], [900, 4000], 4, 1024, None), ([4], [3000], 4, 1000, None), ([150], [1200], 150, 1100, None),
]


@gpu
@pytest.mark.parametrize("n,lens,max_rows,max_keys,rows", PAGED)
@pytest.mark.parametrize("causal", [True, False])
def test_paged(device, n, lens, max_rows, max_keys, rows, causal):
    c = Paged(len(n) + max_rows, lens, 2, 64, 16)
    q = torch.randn((sum(n), 4, 64), generator=torch.Generator().manual_seed(1)).half()
    want, tol = reference(q, c.k, c.v, n, lens, 0.125, causal, [set(range(max_keys, x)) for x in lens])
    rows = sum(n) + 1 if rows is None else rows
    x = torch.zeros((rows, 4, 64), dtype=torch.float16)
    x[: sum(n)] = q[:rows]
    k_pool, v_pool, table, on_lens = c.on_gpu()
    # (the table may be wider than max_keys positions)
    for workspace in (True, False):
        out = torch.full(x.shape, 7.0, dtype=torch.float16, device="cuda")
        attend_paged(device, paged_desc(c.cache, 4, rows, max_rows, min(max_keys, c.width * 16), causal, 0.125), x.cuda(), k_pool, v_pool, table, on_lens, starts_of(n).cuda(), out, workspace)
        compare(out, want, tol, kept_rows(n, max_rows, rows), (n, lens, workspace))


@gpu
@pytest.mark.parametrize("n,lens,max_rows,max_keys,rows,kv_rows", [
    ([100], None, 60, 60, None, None), ([100], None, 60, 100, None, None), ([130, 7, 300], None, 128, 200, None, None), ([40, 60], None, 60, 60, 70, 100), ([90, 33], [200, 40], 50, 210, None, None),
    ([90, 33], [200, 40], 50, 120, None, None), ([40, 60], [80, 90], 60, 90, None, 150), ([700, 300], None, 300, 300, None, None), ([64], [3000], 40, 3000, None, None),
])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(device, n, lens, max_rows, max_keys, rows, kv_rows, causal):
    keys = n if lens is None else lens
    gen = torch.Generator().manual_seed(len(n) + max_rows)
    q = torch.randn((sum(n), 4, 64), generator=gen).half()
    k, v = (torch.randn((sum(keys), 2, 64), generator=gen).half() for _ in range(2))
    rows, kv_rows = sum(n) if rows is None else rows, sum(keys) if kv_rows is None else kv_rows
    first = [sum(keys[:i]) for i in range(len(keys))]
    hidden = [set(range(max_keys, x)) | set(range(max(0, kv_rows - a), x)) for a, x in zip(first, keys)]
    want, tol = reference(q, list(torch.split(k, keys)), list(torch.split(v, keys)), n, keys, 0.125, causal, hidden)
    out = torch.full((rows, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    kv_starts = None if lens is None and rows == kv_rows else starts_of(keys).cuda()
    attend_packed(device, packed_desc(len(n), 4, 2, 64, rows, kv_rows, max_rows, max_keys, causal, 0.125), q[:rows].cuda(), k[:kv_rows].cuda(), v[:kv_rows].cuda(), starts_of(n).cuda(), kv_starts, out)
    compare(out, want, tol, kept_rows(n, max_rows, rows), (n, keys))


@gpu
@pytest.mark.parametrize("heads,kv", [(32, 1), (33, 1), (40, 1), (64, 1), (71, 1), (130, 2), (129, 1)])
@pytest.mark.parametrize("lens", [[1], [37, 128, 0, 129], [3000, 5], [600] * 30], ids=lambda x: f"{len(x)}x{max(x)}")
def test_one_row_of_many_heads_on_one(device, heads, kv, lens):
    """A token of more than 32 heads that share their keys: on both sides of the border between the kernels, and of a tile's."""
    c = Paged(heads, lens, kv, 64, 16)
    q = torch.randn((len(lens), heads, 64), generator=torch.Generator().manual_seed(2)).half()
    want, tol = reference(q, c.k, c.v, [1] * len(lens), lens, 0.125, True)
    k_pool, v_pool, table, on_lens = c.on_gpu()
    for starts in (None, starts_of([1] * len(lens)).cuda()):
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
        attend_paged(device, paged_desc(c.cache, heads, len(lens), 1, c.width * 16, True, 0.125), q.cuda(), k_pool, v_pool, table, on_lens, starts, out)
        close(out, want, tol, (heads, kv, lens))
