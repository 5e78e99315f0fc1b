"""Module harness over the operators: the reference's `Linear` (crates/ratchet-nn/src/linear.rs), its
key/value cache (crates/ratchet-nn/src/kv_cache.rs) and the two blocks of a Phi-2 decoder layer that the
operators of this library cover end to end (crates/ratchet-models/src/phi2/mlp.rs, phi2/attn.rs).
Normalisation, rotary embedding and the residual adds of the layer are other operators and not part of it."""
from typing import List, Optional, Sequence

from . import _ffi
from .tensor import Device, DType, OperationError, Sequences, Tensor


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


class PagedKVEntry:
    """One layer's pools of a PagedKVCache."""

    def __init__(self, owner: "PagedKVCache", k_pool: Tensor, v_pool: Tensor):
        self.owner, self.k_pool, self.v_pool = owner, k_pool, v_pool


class PagedKVCache:
    """A key/value cache whose memory goes to sequences a page at a time (no counterpart in the reference, whose KVEntry reserves the whole capacity,
    kv_cache.rs:3-19): pools [pages, kv_heads, page_size, head_dim] for each layer, and one table for all of them.  `batch` sequences of up to `max_pages` pages.

    A pass over the model: extend(rows) with the new rows of each sequence (a prompt's length, 1 for a step, 0 for none), then the layers with the packed rows, resolved
    before the next extend() or release(): operators of an earlier pass are refused.  What the GPU reads (table, lens, starts) stays in the same memory, so that a pass captured
    into a graph (resolve(wait=False)) runs on what the last extend() left there: on sequences that have grown to any length, in all of no more rows than the
    captured tensors have, and none of a sequence more than the longest had there."""

    def __init__(self, n_layers: int, shape, device: Device, batch: int, max_pages: int):
        import torch
        self.pages, self.kv_heads, self.page_size, self.head_dim = map(int, shape)
        self.layers = [PagedKVEntry(self, Tensor.empty_cache(shape, device, DType.F16), Tensor.empty_cache(shape, device, DType.F16)) for _ in range(n_layers)]
        self.batch, self.max_pages = int(batch), int(max_pages)
        self.free = list(range(self.pages))[::-1]
        self.owned: List[List[int]] = [[] for _ in range(self.batch)]
        self.entries = [0] * self.batch
        self.passes = 0   # what has changed the tensors below, so many times
        where = device.torch_device()
        self.table = torch.full((self.batch, self.max_pages), -1, dtype=torch.int32, device=where)
        self.lens = torch.zeros(self.batch, dtype=torch.int32, device=where)
        self.starts = torch.zeros(self.batch + 1, dtype=torch.int32, device=where)

    def __getitem__(self, i: int) -> PagedKVEntry:
        return self.layers[i]

    def extend(self, rows: Sequence[int]) -> Sequences:
        """Pages for that many new rows of each sequence -> what the operators of the pass take.  An error leaves the cache as it was."""
        import torch
        rows = [int(r) for r in rows]
        if len(rows) != self.batch or any(r < 0 for r in rows):
            raise OperationError(_ffi.RT_ERR_INVALID_SHAPE, f"cache: rows of {self.batch} sequences, got {rows}")
        needs = [-(-(n + r) // self.page_size) - len(own) for n, r, own in zip(self.entries, rows, self.owned)]
        if any(len(own) + n > self.max_pages for own, n in zip(self.owned, needs)) or sum(needs) > len(self.free):
            raise OperationError(_ffi.RT_ERR_OOM, f"cache: {sum(needs)} pages wanted, {len(self.free)} free, {self.max_pages} a sequence")
        self.passes += 1
        for i, (r, n) in enumerate(zip(rows, needs)):
            self.owned[i] += [self.free.pop() for _ in range(n)]
            self.entries[i] += r
        if any(needs):
            self.table.copy_(torch.tensor([own + [-1] * (self.max_pages - len(own)) for own in self.owned], dtype=torch.int32))
        at = [0]
        for r in rows:
            at.append(at[-1] + r)
        self.starts.copy_(torch.tensor(at, dtype=torch.int32))
        self.lens.copy_(torch.tensor(self.entries, dtype=torch.int32))
        return Sequences(self.batch, self.starts, max(rows + [0]), self.lens, self.table, max(self.entries + [0]), self)

    def release(self, i: int):
        """Sequence i has ended: its pages are free."""
        self.passes += 1
        self.free += self.owned[i][::-1]
        self.owned[i], self.entries[i] = [], 0
        self.table[i].fill_(-1)
        self.lens[i] = 0


class SelfAttention:
    """phi2/attn.rs:100-156 without the rotary embedding (another operator): q, k, v projections, the new
    keys and values written into the cache, causal attention over the cached rows, output projection.
    The reference's view / permute / Cache-copy / matmul / softmax / matmul chain is three enqueues here:
    two cache writes that read the projections where they lie, and one attention kernel that reads the
    cache in place and writes [batch, len, heads * head_dim]."""

    def __init__(self, q: Linear, k: Linear, v: Linear, o: Linear, n_heads: int):
        self.q, self.k, self.v, self.o, self.n_heads = q, k, v, o, n_heads

    def schedule(self, input: Tensor, cache=None, sequences: Optional[Sequences] = None) -> Tensor:
        """cache: a KVEntry, and input [b, len, width]; or a PagedKVEntry with the sequences that its cache's extend() gave, and input [1, rows, width], packed.  Sequences
        without a cache: packed prompts that see themselves."""
        q, k, v = self.q.schedule(input), self.k.schedule(input), self.v.schedule(input)   # [b, len, heads * d]
        if isinstance(cache, PagedKVEntry):
            if sequences is None:
                raise OperationError(_ffi.RT_ERR_INVALID_ARG, "attention: a cache in pages needs the pass's sequences")
            if sequences.cache is not None and sequences.cache is not cache.owner:
                raise OperationError(_ffi.RT_ERR_INVALID_ARG, "attention: sequences of another cache")
            keys, values = cache.k_pool.cache_write_paged(k, sequences), cache.v_pool.cache_write_paged(v, sequences)
            return self.o.schedule(q.attention_paged(keys, values, sequences))
        if sequences is not None:
            if cache is not None:
                raise OperationError(_ffi.RT_ERR_UNSUPPORTED, "attention: sequences of different lengths need a cache in pages")
            return self.o.schedule(q.attention_packed(k, v, sequences, self.n_heads))
        B, L, HD = q.shape
        if cache is None:
            cache = KVEntry.allocate((B, self.n_heads, L, HD // self.n_heads), input.device, input.dt)
        offset = cache.entries
        keys = cache.k_cache.cache_write(k, offset)
        values = cache.v_cache.cache_write(v, offset)
        a = q.attention(keys, values, causal=True, kv_len=offset + L, merge_heads=True)
        return self.o.schedule(a)
