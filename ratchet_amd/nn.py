"""Module harness over the operators: the reference's `Linear` (crates/ratchet-nn/src/linear.rs), its
key/value cache (crates/ratchet-nn/src/kv_cache.rs) and the two blocks of a Phi-2 decoder layer that the
operators of this library cover end to end (crates/ratchet-models/src/phi2/mlp.rs, phi2/attn.rs).
Normalisation, rotary embedding and the residual adds of the layer are other operators and not part of it."""
from typing import List, Optional

from .tensor import Device, DType, Tensor


class Linear:
    """linear.rs:9-24: y = x W^T + b as `W.gemm(x, b, false, true, true)`; W may be quantized."""

    def __init__(self, w: Tensor, b: Optional[Tensor] = None):
        self.w, self.b = w, b

    def schedule(self, input: Tensor) -> Tensor:
        b = self.b.cast(input.dt) if self.b is not None else None   # linear.rs:18-22
        return self.w.gemm(input, b, False, True, True)


class MLP:
    """phi2/mlp.rs:6-16: fc2(gelu(fc1(x))).  The activation runs in fc1's epilogue."""

    def __init__(self, fc1: Linear, fc2: Linear):
        self.fc1, self.fc2 = fc1, fc2

    def schedule(self, input: Tensor) -> Tensor:
        return self.fc2.schedule(self.fc1.schedule(input).gelu())


class KVEntry:
    """kv_cache.rs:3-19: one layer's key and value caches [batch, heads, capacity, head_dim] and the rows in use.
    With dt = DType.Q4_0 they are held in 4-bit blocks, and may have fewer heads than the queries (heads a multiple of them)."""

    def __init__(self, k_cache: Tensor, v_cache: Tensor, entries: int = 0):
        self.k_cache, self.v_cache, self.entries = k_cache, v_cache, entries

    @staticmethod
    def allocate(shape, device: Device, dt: DType = DType.F16) -> "KVEntry":
        return KVEntry(Tensor.empty_cache(shape, device, dt), Tensor.empty_cache(shape, device, dt), 0)


class KVCache:
    """kv_cache.rs:21-58."""

    def __init__(self, n_layers: int, shape, device: Device, dt: DType = DType.F16):
        self.layers: List[KVEntry] = [KVEntry.allocate(shape, device, dt) for _ in range(n_layers)]

    def __getitem__(self, i: int) -> KVEntry:
        return self.layers[i]

    def update(self, offset: int):
        for e in self.layers:
            e.entries += offset

    def entries(self, layer: int) -> int:
        return self.layers[layer].entries

    def reset(self):
        for e in self.layers:
            e.entries = 0


class SelfAttention:
    """phi2/attn.rs:100-156 without the rotary embedding (another operator): q, k, v projections, the new
    keys and values written into the cache, causal attention over the cached rows, output projection.
    The reference's view / permute / Cache-copy / matmul / softmax / matmul chain is three enqueues here:
    two cache writes that read the projections where they lie, and one attention kernel that reads the
    cache in place and writes [batch, len, heads * head_dim]."""

    def __init__(self, q: Linear, k: Linear, v: Linear, o: Linear, n_heads: int):
        self.q, self.k, self.v, self.o, self.n_heads = q, k, v, o, n_heads

    def schedule(self, input: Tensor, cache: Optional[KVEntry] = None) -> Tensor:
        q, k, v = self.q.schedule(input), self.k.schedule(input), self.v.schedule(input)   # [b, len, heads * d]
        B, L, HD = q.shape
        if cache is None:
            cache = KVEntry.allocate((B, self.n_heads, L, HD // self.n_heads), input.device, input.dt)
        offset = cache.entries
        keys = cache.k_cache.cache_write(k, offset)
        values = cache.v_cache.cache_write(v, offset)
        a = q.attention(keys, values, causal=True, kv_len=offset + L, merge_heads=True)
        return self.o.schedule(a)
