"""Passes over a nn.PagedKVCache: a pass whose sequences are no longer the cache's last is refused, and a captured pass runs on what the last extend() left, however far the sequences
have grown."""
import numpy as np
import pytest
import torch

from ragged_cases import close, reference
from ratchet_amd import Device, OperationError, Sequences, Tensor, nn

CPU = Device.CPU
gpu = pytest.mark.gpu


def zeros(*shape, dt=np.float16):
    return Tensor.from_data(np.zeros(shape, dt))


@pytest.mark.parametrize("then", ["extend", "release"])
def test_operators_of_an_earlier_pass_are_refused(then):
    """What they would read is the later pass's: the lengths, starts and table are the cache's own."""
    c = nn.PagedKVCache(1, (6, 2, 16, 64), CPU, 2, 3)
    old = c.extend([3, 1])
    c.extend([1, 1]) if then == "extend" else c.release(1)
    with pytest.raises(OperationError, match="pass"):
        c[0].k_pool.cache_write_paged(zeros(4, 128), old)
    with pytest.raises(OperationError, match="pass"):
        zeros(4, 512).attention_paged(c[0].k_pool, c[0].v_pool, old)
    with pytest.raises(OperationError, match="pass"):
        zeros(4, 512).attention_packed(zeros(4, 128), zeros(4, 128), old, 8)
    new = c.extend([1, 2])
    for bad in ([100, 0], [1]):      # an extend() that fails leaves the pass as it was
        with pytest.raises(OperationError):
            c.extend(bad)
    assert zeros(3, 512).attention_paged(c[0].k_pool, c[0].v_pool, new).shape == (3, 512)


def test_sequences_of_another_cache_are_refused():
    a, b = (nn.PagedKVCache(2, (6, 1, 16, 64), CPU, 2, 3) for _ in range(2))
    attn = nn.SelfAttention(*[nn.Linear(zeros(64, 64)) for _ in range(4)], 1)
    a.extend([1, 1])
    other = b.extend([2, 1])
    with pytest.raises(OperationError, match="cache"):
        attn.schedule(zeros(1, 3, 64), a[1], other)
    assert attn.schedule(zeros(1, 3, 64), b[1], other).shape == (1, 3, 64)


def put(t, x):
    t.storage.copy_(x.reshape(-1).view(torch.uint8))


class Numbers:
    """Queries, keys and values of a pass in memory that stays, and what each sequence has been given so far."""

    def __init__(self, device, rows, heads, kv, d, batch, seed):
        self.gen, self.sizes = torch.Generator().manual_seed(seed), ((rows, heads, d), (rows, kv, d), (rows, kv, d))
        self.on = [Tensor.from_data(np.zeros((s[0], s[1] * s[2]), np.float16)).to(device) for s in self.sizes]
        self.keys, self.values = ([torch.zeros((0, kv, d), dtype=torch.float16) for _ in range(batch)] for _ in range(2))

    def draw(self, n):
        """New numbers, of which the first sum(n) rows go to the sequences."""
        q, k, v = (torch.randn(s, generator=self.gen).half() for s in self.sizes)
        for t, x in zip(self.on, (q, k, v)):
            put(t, x)
        at = 0
        for i, r in enumerate(n):
            self.keys[i], self.values[i] = torch.cat([self.keys[i], k[at:at + r]]), torch.cat([self.values[i], v[at:at + r]])
            at += r
        return q[:at]

    def want(self, q, n):
        return reference(q, self.keys, self.values, n, [len(x) for x in self.keys], self.sizes[0][2] ** -0.5, True)


def values_of(t, shape):
    return t.storage.view(torch.float16)[: int(np.prod(shape))].view(*shape)


@gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_a_captured_pass_follows_the_cache(device, rows):
    """Captured where the sequences are short, replayed over 20 extend()s that give pages to all of them, let one rest and end one; eager passes between."""
    batch, heads, kv, d, ps = 3, 8, 2, 64, 16
    cache = nn.PagedKVCache(1, (3 * 60, kv, ps, d), device, batch, 60)
    short = [5, 0, 14]
    x = Numbers(device, sum(short), heads, kv, d, batch, rows)

    def attend(x, seqs, wait):
        q, k, v = x.on
        entry = cache[0]
        return q.attention_paged(entry.k_pool.cache_write_paged(k, seqs), entry.v_pool.cache_write_paged(v, seqs), seqs).resolve(wait)

    def eager(n):
        e = Numbers(device, sum(n), heads, kv, d, batch, 7 + sum(n))
        e.keys, e.values = y.keys, y.values
        q = e.draw(n)
        out = values_of(attend(e, cache.extend(n), True), q.shape)
        close(out, *e.want(q, n), ("eager", n))

    y = x
    q = x.draw(short)
    out = values_of(attend(x, cache.extend(short), True), q.shape)
    close(out, *x.want(q, short), "prompts")
    y = Numbers(device, batch * rows, heads, kv, d, batch, 100 + rows)
    y.keys, y.values = x.keys, x.values
    n = [rows] * batch
    q = y.draw(n)
    seqs = cache.extend(n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        node = attend(y, seqs, False)
    graph.replay()
    torch.cuda.synchronize()
    close(values_of(node, q.shape), *y.want(q, n), "captured")
    for step in range(20):
        n = [rows, 0 if step % 5 == 3 else rows, rows]
        q = y.draw(n)
        cache.extend(n)
        values_of(node, q.shape).fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        close(values_of(node, q.shape), *y.want(q, n), step)
        if step == 9:
            cache.release(1)
            y.keys[1], y.values[1] = y.keys[1][:0], y.values[1][:0]
            eager([1, 33, 0])
    assert max(cache.entries) > 16 * rows and min(len(o) for o in cache.owned) > 1


@gpu
def test_a_captured_module(device):
    """SelfAttention captured with wait=False: the same as the module run pass by pass on a cache of its own."""
    W, H, batch = 256, 4, 3
    rng = np.random.default_rng(0)

    def lin(n, k):
        return nn.Linear(Tensor.from_data((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16)).to(device), Tensor.from_data((0.1 * rng.standard_normal(n)).astype(np.float16)).to(device))
    attn = nn.SelfAttention(lin(W, W), lin(W, W), lin(W, W), lin(W, W), H)
    caches = [nn.PagedKVCache(1, (60, H, 16, W // H), device, batch, 20) for _ in range(2)]
    x = Tensor.from_data(rng.standard_normal((1, 12, W)).astype(np.float16)).to(device)
    for c in caches:
        attn.schedule(x, c[0], c.extend([7, 1, 4])).resolve()
    x = Tensor.from_data(np.zeros((1, batch, W), np.float16)).to(device)
    seqs = [c.extend([1] * batch) for c in caches]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        node = attn.schedule(x, caches[0][0], seqs[0]).resolve(wait=False)
    twin = caches[1]
    bits = lambda t: t.storage[: 2 * batch * W].cpu()
    for step in range(40):
        if step:
            for c in caches:
                c.extend([1] * batch)
        put(x, torch.from_numpy(rng.standard_normal((1, batch, W)).astype(np.float16)))
        graph.replay()
        torch.cuda.synchronize()
        # (the same bounds choose the same kernels, whose results are the same bits)
        want = attn.schedule(x, twin[0], Sequences(batch, twin.starts, 1, twin.lens, twin.table)).resolve()
        assert torch.equal(bits(node), bits(want)), step
        torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("then", ["extend", "release"])
def test_a_pass_run_too_late_is_refused(device, then):
    """Scheduled, and resolved behind the next extend() or a release(): nothing is written, and the pass that is the cache's last runs."""
    kv, d = 2, 64
    c = nn.PagedKVCache(1, (8, kv, 16, d), device, 2, 4)
    n = [3, 1]
    x = Numbers(device, 4, 4, kv, d, 2, 1)
    q0 = x.draw(n)
    seqs = c.extend(n)
    q, k, v = x.on
    late = q.attention_paged(c[0].k_pool.cache_write_paged(k, seqs), c[0].v_pool.cache_write_paged(v, seqs), seqs)
    write = c[0].k_pool.cache_write_paged(k, seqs)
    packed = q.attention_packed(k, v, seqs, 4)
    c.extend([1, 1]) if then == "extend" else c.release(1)
    for node in (late, write, packed):
        with pytest.raises(OperationError, match="pass"):
            node.resolve()
    torch.cuda.synchronize()
    assert not bool(c[0].k_pool.storage.any()) and not bool(c[0].v_pool.storage.any())
    assert q0.shape[0] == 4


@gpu
@pytest.mark.parametrize("k_type,v_type", [(np.float32, np.float32), (np.float32, np.float16), (np.float16, np.float32)])
def test_writes_of_f32_rows(device, k_type, v_type):
    """Keys and values of either type, in one launch where they are of one: the rows rounded to f16, bit for bit, and what the attention then reads."""
    kv, d, ps = 2, 64, 16
    c = nn.PagedKVCache(1, (6, kv, ps, d), device, 2, 4)
    rng = np.random.default_rng(3)
    for n in ([20, 3], [1, 14]):
        seqs = c.extend(n)
        k, v = ((rng.standard_normal((sum(n), kv * d)) * 3).astype(t) for t in (k_type, v_type))
        q = rng.standard_normal((sum(n), kv * d)).astype(np.float16)
        K, V, Q = (Tensor.from_data(x).to(device) for x in (k, v, q))
        before = [p.to(CPU).storage.copy() for p in (c[0].k_pool, c[0].v_pool)]
        out = Q.attention_paged(c[0].k_pool.cache_write_paged(K, seqs), c[0].v_pool.cache_write_paged(V, seqs), seqs).resolve()
        table, want, at = c.table.cpu().numpy(), before, 0
        for i, r in enumerate(n):
            for j in range(r):
                p = c.entries[i] - r + j
                for pool, x in zip(want, (k, v)):
                    pool[table[i, p // ps], :, p % ps] = x[at + j].astype(np.float16).reshape(kv, d)
            at += r
        for pool, x in zip((c[0].k_pool, c[0].v_pool), want):
            assert np.array_equal(pool.to(CPU).storage.view(np.uint16), x.view(np.uint16))
        held = [[torch.from_numpy(x[table[i, : -(-m // ps)]].transpose(0, 2, 1, 3).reshape(-1, kv, d)[:m].copy()) for i, m in enumerate(c.entries)] for x in want]
        exact = reference(torch.from_numpy(q).view(-1, kv, d), *held, n, c.entries, d ** -0.5, True)
        close(values_of(out, (sum(n), kv, d)), *exact)
