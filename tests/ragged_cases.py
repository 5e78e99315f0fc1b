"""What the tests of packed sequences and paged caches share: inputs, the operators in 64 bits, how far an output may be off, and the calls.

attention  out = sum_j p~_j v_j / sum_j p~_j in the kernels, p~ the probabilities rounded to f16 (half a step: 2^-11 relative), then rounded to f16.  With p the exact
           ones, w_j = p_j / sum p and spread = sum_j w_j |v_j - out|:
             rounding of p                    2^-11 spread
             a score off by e (relative to p) 2 e spread, e = (D + 8) 2^-24 scale max_j sum_c |q_c k_jc|, and 2^-21 for the exponential and its argument
             sums of N terms in f32           N 2^-24 sum_j w_j |v_j|
             the output                       2^-11 |out|, and 2^-25 where it is subnormal
           A probability below 2^-31 of the largest may be lost whole: 2^-31 N max |v|.
"""
import ctypes
import math

import torch

from ratchet_amd import _ffi


def table_of(lens, page_size, pages, width, gen, spare=0):
    """Pages given out in any order; -1 where a sequence has none.  The lists of pages do not overlap."""
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range((n + page_size - 1) // page_size + spare):
            if j < width:
                table[i, j] = order.pop()
    return table


def starts_of(sizes):
    return torch.tensor([0] + torch.tensor(sizes, dtype=torch.int64).cumsum(0).tolist() if len(sizes) else [0], dtype=torch.int32)


def reference(q, k, v, n, lens, scale, causal, hidden=None):
    """q [rows, H, D], k, v: a list of [keys, KV, D] per sequence; n rows and lens keys of each -> (out, tolerance), f64 [rows, H, D].  hidden: per sequence a
    set of positions that nobody sees."""
    q = q.double()
    out, tol = torch.full(q.shape, float("nan"), dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    at = 0
    for b, (rows, keys) in enumerate(zip(n, lens)):
        kb, vb = k[b].double()[:keys], v[b].double()[:keys]
        g = q.shape[1] // kb.shape[1] if kb.shape[1] else 1
        for h in range(q.shape[1]):
            x, y, z = q[at:at + rows, h], kb[:, h // g], vb[:, h // g]
            seen = torch.arange(keys)[None, :] <= (torch.arange(rows)[:, None] + keys - rows if causal else keys)
            if hidden is not None and len(hidden[b]):
                seen = seen.clone()
                seen[:, torch.tensor(sorted(hidden[b]))] = False
            s = torch.where(seen, scale * torch.nan_to_num(x @ y.T, 0.0, 0.0, 0.0), float("-inf"))
            m = s.amax(-1, keepdim=True) if keys else torch.zeros((rows, 1))
            p = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
            w = p / p.sum(-1, keepdim=True)
            zz = torch.nan_to_num(z, 0.0, 0.0, 0.0)     # what is not finite is checked apart
            o = w @ zz
            off = x.shape[1] + 8
            e = off * 2.0**-24 * abs(scale) * (x.abs() @ torch.nan_to_num(y, 0.0, 0.0, 0.0).abs().T * seen).amax(-1) if keys else torch.zeros(rows, dtype=torch.float64)
            spread = torch.stack([(w * (zz[None, :, c] - o[:, None, c]).abs()).sum(-1) for c in range(z.shape[1])], -1) if keys else torch.zeros_like(o)
            out[at:at + rows, h] = o if keys else float("nan")
            big = zz.abs().max() if keys else 0.0
            tol[at:at + rows, h] = (2.0**-11 + 2 * e[:, None] + 2.0**-20) * spread + keys * 2.0**-24 * (w @ zz.abs()) + 2.0**-11 * o.abs() + 2.0**-25 + 2.0**-31 * keys * big
        at += rows
    return out, tol


def close(got, want, tol, what=""):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN in other places", int(torch.isnan(got).sum()), int(torch.isnan(want).sum()))
    ok = torch.isnan(want) | ((got - want).abs() <= tol)
    if not bool(ok.all()):
        i = int(torch.where(ok, 0.0, ((got - want).abs() / tol)).argmax())
        raise AssertionError((what, "row, head, dimension", [int(x) for x in torch.unravel_index(torch.tensor(i), want.shape)], got.flatten()[i].item(),
                              want.flatten()[i].item(), tol.flatten()[i].item(), "of them off", int((~ok).sum())))


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def packed_desc(batch, heads, kv_heads, head_dim, rows, kv_rows, max_rows, max_keys, causal, scale, q_strides=None, k_strides=None, v_strides=None, o_strides=None):
    d = _ffi.AttentionPackedDesc()
    d.batch, d.heads, d.kv_heads, d.head_dim, d.rows, d.kv_rows = batch, heads, kv_heads, head_dim, rows, kv_rows
    d.max_rows, d.max_keys, d.causal, d.scale = max_rows, max_keys, int(causal), scale
    d.q_strides[:] = q_strides or [heads * head_dim, head_dim]
    d.k_strides[:] = k_strides or [kv_heads * head_dim, head_dim]
    d.v_strides[:] = v_strides or [kv_heads * head_dim, head_dim]
    d.o_strides[:] = o_strides or [heads * head_dim, head_dim]
    return d


def cache_desc(batch, kv_heads, head_dim, pages, page_size, table_width, table_stride=None):
    c = _ffi.PagedCacheDesc()
    c.batch, c.kv_heads, c.head_dim, c.pages, c.page_size = batch, kv_heads, head_dim, pages, page_size
    c.table_width, c.table_stride = table_width, table_width if table_stride is None else table_stride
    return c


def paged_desc(cache, heads, rows, max_rows, max_keys, causal, scale, q_strides=None, o_strides=None):
    d = _ffi.AttentionPagedDesc()
    d.cache, d.heads, d.rows, d.max_rows, d.max_keys, d.causal, d.scale = cache, heads, rows, max_rows, max_keys, int(causal), scale
    d.q_strides[:] = q_strides or [heads * cache.head_dim, cache.head_dim]
    d.o_strides[:] = o_strides or [heads * cache.head_dim, cache.head_dim]
    return d


def workspace_for(ask, desc, fill=0xFF):
    need = ctypes.c_uint64()
    assert ask(desc, need) == _ffi.RT_OK
    return torch.full((need.value,), fill, dtype=torch.uint8, device="cuda") if need.value else None


def attend_packed(device, desc, q, k, v, starts, kv_starts, out, workspace=True):
    L = _ffi.lib()
    ws = workspace_for(L.rt_attention_packed_workspace_bytes, desc) if workspace is True else workspace if workspace is not False else None
    st = L.rt_attention_packed_enqueue(device.ctx, desc, ptr(q), ptr(k), ptr(v), ptr(starts), ptr(kv_starts), ptr(out), ptr(ws), 0 if ws is None else ws.numel(), stream())
    assert st == _ffi.RT_OK, (_ffi.status_string(st), L.rt_last_error(device.ctx))
    return out


def attend_paged(device, desc, q, k_pool, v_pool, table, lens, starts, out, workspace=True):
    L = _ffi.lib()
    ws = workspace_for(L.rt_attention_paged_workspace_bytes, desc) if workspace is True else workspace if workspace is not False else None
    st = L.rt_attention_paged_enqueue(device.ctx, desc, ptr(q), ptr(k_pool), ptr(v_pool), ptr(table), ptr(lens), ptr(starts), ptr(out), ptr(ws),
                                      0 if ws is None else ws.numel(), stream())
    assert st == _ffi.RT_OK, (_ffi.status_string(st), L.rt_last_error(device.ctx))
    return out


def write_paged(device, cache, k_pool, k, v_pool, v, table, lens, starts, rows, strides=None):
    L = _ffi.lib()
    st = L.rt_cache_write_paged_enqueue(device.ctx, cache, _ffi.RT_F16 if k.dtype == torch.float16 else _ffi.RT_F32, ptr(k_pool), ptr(k), ptr(v_pool), ptr(v),
                                        (ctypes.c_int64 * 2)(*(strides or [cache.kv_heads * cache.head_dim, cache.head_dim])), ptr(table), ptr(lens), ptr(starts), rows, stream())
    assert st == _ffi.RT_OK, (_ffi.status_string(st), L.rt_last_error(device.ctx))


class Paged:
    """Keys and values of some sequences in pages that are given out in any order; what no sequence has is NaN."""

    def __init__(self, seed, lens, kv_heads, head_dim, page_size, max_keys=None, spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.page_size = lens, page_size
        most = max(list(lens) + [1]) if max_keys is None else max_keys
        self.width = (most + page_size - 1) // page_size
        pages = sum((n + page_size - 1) // page_size for n in lens) + 2
        self.table = table_of(lens, page_size, pages, self.width, gen)
        self.k = [spread * torch.randn((n, kv_heads, head_dim), generator=gen) for n in lens]
        self.v = [torch.randn((n, kv_heads, head_dim), generator=gen) for n in lens]
        self.k, self.v = [x.half() for x in self.k], [x.half() for x in self.v]
        self.k_pool, self.v_pool = (torch.full((pages, kv_heads, page_size, head_dim), float("nan"), dtype=torch.float16) for _ in range(2))
        self.fill()
        self.cache = cache_desc(len(lens), kv_heads, head_dim, pages, page_size, self.width)

    def fill(self):
        for pool, rows in ((self.k_pool, self.k), (self.v_pool, self.v)):
            for i, x in enumerate(rows):
                p = torch.arange(x.shape[0])
                page = self.table[i].long()[p // self.page_size]
                ok = page >= 0
                pool[page[ok], :, (p % self.page_size)[ok]] = x[ok]

    def on_gpu(self):
        return [x.cuda() for x in (self.k_pool, self.v_pool, self.table, torch.tensor(self.lens, dtype=torch.int32))]
