"""The Python calls on sequences of different lengths: the modules with a cache in pages against the same modules sequence by sequence, graph order, refusals."""
import numpy as np
import pytest
import torch

from ratchet_amd import DType, Device, InvariantError, OperationError, Sequences, Tensor, nn

CPU = Device.CPU
gpu = pytest.mark.gpu


def zeros(*shape, dt=np.float16):
    return Tensor.from_data(np.zeros(shape, dt))


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def fine():
    return Sequences(2, ints(0, 3, 4), 3, ints(5, 6), torch.zeros((2, 4), dtype=torch.int32))


def test_shapes_without_a_device():
    pool, seqs = Tensor.empty_cache((6, 2, 16, 64), CPU), fine()
    assert pool.cache_write_paged(zeros(4, 128), seqs).shape == (6, 2, 16, 64)
    assert pool.cache_write_paged(zeros(1, 4, 128, dt=np.float32), seqs).shape == (6, 2, 16, 64)
    q = zeros(1, 4, 512)
    assert q.attention_paged(pool, pool, seqs).shape == (1, 4, 512)
    assert q.attention_packed(zeros(4, 128), zeros(4, 128), seqs, 8).shape == (1, 4, 512)
    assert q.attention_paged(pool, pool, seqs).op.desc.max_keys == 64


@pytest.mark.parametrize("change", [
    dict(starts=ints(0, 3)), dict(starts=torch.zeros(3)), dict(lens=ints(5)), dict(lens=None), dict(table=None), dict(table=ints(0, 0)), dict(table=torch.zeros((3, 4), dtype=torch.int32)),
    dict(table=torch.zeros((4, 2), dtype=torch.int32).t()), dict(starts=None, max_rows=3),
])
def test_refused_sequences(change):
    args = dict(batch=2, starts=ints(0, 3, 4), max_rows=3, lens=ints(5, 6), table=torch.zeros((2, 4), dtype=torch.int32))
    seqs = Sequences(**{**args, **change})
    pool, q = Tensor.empty_cache((6, 2, 16, 64), CPU), zeros(4, 512)
    with pytest.raises(OperationError):
        pool.cache_write_paged(zeros(4, 128), seqs)
    with pytest.raises(OperationError):
        q.attention_paged(pool, pool, seqs)


def test_refusals():
    pool, seqs = Tensor.empty_cache((6, 2, 16, 64), CPU), fine()
    with pytest.raises(OperationError):
        Sequences(1 << 32)
    with pytest.raises(OperationError):
        Sequences(2, max_rows=-1)
    with pytest.raises(OperationError):
        pool.cache_write_paged(zeros(4, 64), seqs)                                    # rows of another width
    with pytest.raises(InvariantError):
        Tensor.empty_cache((6, 2, 24, 64), CPU).cache_write_paged(zeros(4, 128), seqs)  # pages of 24
    with pytest.raises(InvariantError):
        Tensor.empty_cache((6, 2, 16, 64), CPU, DType.F32).cache_write_paged(zeros(4, 128), seqs)
    with pytest.raises(OperationError):
        zeros(4, 500).attention_paged(pool, pool, seqs)
    with pytest.raises(OperationError):
        zeros(4, 192).attention_paged(pool, pool, seqs)                               # 3 heads on 2
    with pytest.raises(InvariantError):
        zeros(4, 512, dt=np.float32).attention_paged(pool, pool, seqs)
    with pytest.raises(OperationError):
        zeros(4, 512).attention_paged(pool, Tensor.empty_cache((6, 2, 32, 64), CPU), seqs)
    with pytest.raises(OperationError):
        zeros(4, 512).attention_paged(pool, pool, Sequences(2, ints(0, 3, 4), 3, ints(5, 6), torch.zeros((2, 4), dtype=torch.int32), max_keys=65))
    with pytest.raises(OperationError):
        zeros(4, 512).attention_packed(zeros(4, 128), zeros(4, 128), seqs, 7)
    with pytest.raises(OperationError):
        zeros(4, 512).attention_packed(zeros(5, 128), zeros(5, 128), seqs, 8)
    with pytest.raises(InvariantError):
        zeros(4, 512).attention_packed(zeros(4, 128, dt=np.float32), zeros(4, 128, dt=np.float32), seqs, 8)
    with pytest.raises(OperationError):
        zeros(4, 512).attention_packed(zeros(4, 128), zeros(4, 128), Sequences(2, None, 3), 8)


def test_pages_are_given_out_and_taken_back():
    c = nn.PagedKVCache(2, (5, 1, 16, 64), CPU, 3, 4)
    s = c.extend([17, 0, 16])
    assert c.entries == [17, 0, 16] and [len(o) for o in c.owned] == [2, 0, 1] and s.max_rows == 17 and s.max_keys == 17
    assert s.starts.tolist() == [0, 17, 17, 33] and s.lens.tolist() == [17, 0, 16]
    assert s.table[0].tolist() == c.owned[0] + [-1, -1] and s.table[1].tolist() == [-1] * 4
    before = (list(c.free), [list(o) for o in c.owned], list(c.entries), c.table.clone(), c.lens.clone())
    for rows in ([1, 1, 33], [64, 0, 0], [1, 1], [-1, 0, 0]):     # more than are free, more than a sequence may have, rows that are none
        with pytest.raises(OperationError):
            c.extend(rows)
        assert (c.free, c.owned, c.entries) == before[:3] and torch.equal(c.table, before[3]) and torch.equal(c.lens, before[4])
    s = c.extend([1, 1, 1])
    assert c.entries == [18, 1, 17] and not c.free and s.starts.tolist() == [0, 1, 2, 3]
    assert sorted(sum(c.owned, [])) == list(range(5))
    c.release(0)
    assert c.entries == [0, 1, 17] and len(c.free) == 2 and s.table[0].tolist() == [-1] * 4 and s.lens.tolist() == [0, 1, 17]
    c.extend([30, 0, 0])
    assert sorted(sum(c.owned, [])) == list(range(5))
    attn = nn.SelfAttention(*[nn.Linear(zeros(64, 64)) for _ in range(4)], 1)
    with pytest.raises(OperationError):
        attn.schedule(zeros(1, 3, 64), c[0])                       # without the pass's sequences
    with pytest.raises(OperationError):
        attn.schedule(zeros(1, 3, 64), nn.KVEntry.allocate((1, 1, 8, 64), CPU), s)


def layer(device, width, kv_width, heads, seed):
    rng = np.random.default_rng(seed)

    def lin(n, k):
        return nn.Linear(Tensor.from_data((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16)).to(device), Tensor.from_data((0.1 * rng.standard_normal(n)).astype(np.float16)).to(device))
    return nn.SelfAttention(lin(width, width), lin(kv_width, width), lin(kv_width, width), lin(width, width), heads)


@gpu
def test_attention_blocks_with_pages_and_packed(device):
    """Prompts of three lengths, then steps with one sequence resting and one that ends: each sequence alone through the contiguous cache gives the same rows."""
    W, H = 256, 4
    attn = layer(device, W, W, H, 0)
    rng = np.random.default_rng(1)
    cache = nn.PagedKVCache(1, (40, H, 16, W // H), device, 3, 20)
    single = [nn.KVCache(1, (1, H, 320, W // H), device) for _ in range(3)]
    run = lambda t: t.resolve().to(Device.CPU).storage
    for rows in ([100, 1, 37], [1, 1, 1], [1, 0, 3], [5, 1, 1]):
        x = [rng.standard_normal((1, r, W)).astype(np.float16) for r in rows]
        seqs = cache.extend(rows)
        X = Tensor.from_data(np.concatenate(x, axis=1)).to(device)
        got = run(attn.schedule(X, cache[0], seqs))
        assert got.shape == (1, sum(rows), W)
        packed = run(attn.schedule(X, sequences=seqs)) if rows[0] == 100 else None
        at = 0
        for i, r in enumerate(rows):
            if r == 0:
                continue
            want = run(attn.schedule(Tensor.from_data(x[i]).to(device), single[i][0]))
            single[i].update(r)
            for a in [got] + ([packed] if packed is not None else []):
                # the same operators on the same numbers, f32 sums in another order
                np.testing.assert_allclose(a[:, at:at + r].astype(np.float32), want.astype(np.float32), rtol=2e-2, atol=4e-3)
            at += r
        if rows == [1, 0, 3]:
            cache.release(0)
            single[0].reset()


@gpu
def test_shared_heads(device):
    """Fewer heads of keys than of queries, f32 sources: as the operator on the projections."""
    W, H, KV = 256, 8, 2
    D = W // H
    attn = layer(device, W, KV * D, H, 3)
    rng = np.random.default_rng(4)
    cache = nn.PagedKVCache(1, (30, KV, 16, D), device, 2, 10)
    keys, values = [np.zeros((0, KV, D), np.float16) for _ in range(2)], [np.zeros((0, KV, D), np.float16) for _ in range(2)]
    for rows in ([40, 9], [1, 1]):
        x = rng.standard_normal((1, sum(rows), W)).astype(np.float16)
        seqs = cache.extend(rows)
        X = Tensor.from_data(x).to(device)
        got = attn.schedule(X, cache[0], seqs).resolve().to(Device.CPU).storage
        q, k, v = (m.schedule(X).resolve().to(Device.CPU).storage[0] for m in (attn.q, attn.k, attn.v))
        at, want = 0, np.zeros((sum(rows), W))
        for i, r in enumerate(rows):
            keys[i] = np.concatenate([keys[i], k[at:at + r].reshape(r, KV, D)])
            values[i] = np.concatenate([values[i], v[at:at + r].reshape(r, KV, D)])
            n = keys[i].shape[0]
            hidden = np.arange(n)[None] > np.arange(r)[:, None] + n - r
            for h in range(H):
                s = q[at:at + r, h * D:(h + 1) * D].astype(np.float64) @ keys[i][:, h // 4].astype(np.float64).T / np.sqrt(D)
                p = np.exp(np.where(hidden, -np.inf, s - s.max(-1, keepdims=True)))
                want[at:at + r, h * D:(h + 1) * D] = p / p.sum(-1, keepdims=True) @ values[i][:, h // 4].astype(np.float64)
            at += r
        out = attn.o.schedule(Tensor.from_data(want.astype(np.float16)[None]).to(device)).resolve().to(Device.CPU).storage
        np.testing.assert_allclose(got.astype(np.float32), out.astype(np.float32), rtol=2e-2, atol=4e-3)


@gpu
def test_order_of_the_two_writes(device):
    """Keys and values written by one launch only where that cannot be told from one after the other."""
    kv, d, ps = 2, 64, 16
    seqs = Sequences(1, None, 3, torch.tensor([3], dtype=torch.int32).cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda())
    other = Sequences(1, None, 3, torch.tensor([20], dtype=torch.int32).cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda())
    rng = np.random.default_rng(5)
    a, b = (rng.standard_normal((3, kv * d)).astype(np.float16) for _ in range(2))
    q = Tensor.from_data(rng.standard_normal((3, kv * d)).astype(np.float16)).to(device)

    def place(pool, x, n):
        for i in range(3):
            p = n - 3 + i
            pool[[1, 0][p // ps], :, p % ps] = x[i].reshape(kv, d)

    for case in ("two pools", "one pool", "other lengths"):
        K = Tensor.empty_cache((2, kv, ps, d), device)
        V = K if case == "one pool" else Tensor.empty_cache((2, kv, ps, d), device)
        A, B = Tensor.from_data(a).to(device), Tensor.from_data(b).to(device)
        keys, values = K.cache_write_paged(A, seqs), V.cache_write_paged(B, other if case == "other lengths" else seqs)
        q.attention_paged(keys, values, seqs).resolve()
        wk, wv = np.zeros((2, kv, ps, d), np.float16), np.zeros((2, kv, ps, d), np.float16)
        place(wk, a, 3)
        place(wk if case == "one pool" else wv, b, 20 if case == "other lengths" else 3)
        assert np.array_equal(K.to(Device.CPU).storage, wk), case
        if case != "one pool":
            assert np.array_equal(V.to(Device.CPU).storage, wv), case
