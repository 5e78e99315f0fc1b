"""The operators that serve sequences of different lengths together: the write into a key/value cache held in pages, the attention that
reads such a cache, and the attention of whole prompts that lie packed one behind another.

Sequence b of a batch has the query rows starts[b] .. starts[b + 1] - 1 of one packed tensor.

A paged cache is a pool [pages, kv_heads, page_size, head_dim] for keys and one for values, and a table: entry j of a sequence's row is the page that
holds its positions j * page_size .. (j + 1) * page_size - 1.  lens[b] positions of sequence b are in use; its new rows are the last of them.

  write      the new rows of every sequence, packed, into both pools; the pools come back.  rows = 1 is a decode step, more are prompts.
  paged      query rows against the pages of their sequences, heads / kv_heads query heads on one head of keys.  rows = 1 is a decode step, a few
             are drafted tokens, many a prompt, or a part of one behind what is cached of it.
  packed     prompts packed [rows, (heads + 2 kv_heads) * head_dim] as a fused projection leaves them, each of which sees itself alone: causal, or whole
             as an encoder does.

Shapes: the head sizes and lengths of this repository's tests and benchmark (heads of 64, 80, 96 and 128, 1500 frames of an encoder's six heads of 64) and
generic ones around them; pages of 16 to 256 positions.
"""
import math

import torch

own = False

GPU = "cuda:0"


def listed():
    return [
        # a decode step of 32 sequences: latency
        {"name": "write_1", "kind": "write", "batch": 32, "kv_heads": 8, "head_dim": 128, "page_size": 16, "rows": 1, "before": 200, "source": "f16"},
        # a batch of prompts of different lengths
        {"name": "write_2048", "kind": "write", "batch": 8, "kv_heads": 24, "head_dim": 96, "page_size": 64, "rows": 2048, "before": 37, "source": "f32"},
        # one sequence with 1024 positions behind it, a head of keys for each of queries: latency
        {"name": "paged_1", "kind": "paged", "batch": 1, "heads": 32, "kv_heads": 32, "head_dim": 80, "page_size": 16, "rows": 1, "keys": 1024, "ragged": False},
        # one long conversation, four query heads on a head of keys
        {"name": "paged_long", "kind": "paged", "batch": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "page_size": 16, "rows": 1, "keys": 32768, "ragged": False},
        # a serving batch of sequences of different lengths: the most bytes
        {"name": "paged_batch", "kind": "paged", "batch": 32, "heads": 32, "kv_heads": 8, "head_dim": 128, "page_size": 16, "rows": 1, "keys": 8192, "ragged": True},
        # drafted tokens of a few sequences
        {"name": "paged_7", "kind": "paged", "batch": 4, "heads": 24, "kv_heads": 24, "head_dim": 96, "page_size": 32, "rows": 7, "keys": 2001, "ragged": True},
        # parts of prompts behind what is cached of them
        {"name": "paged_512", "kind": "paged", "batch": 2, "heads": 32, "kv_heads": 8, "head_dim": 128, "page_size": 64, "rows": 512, "keys": 4096, "ragged": True},
        # many short prompts at once: latency, and rows of several sequences beside each other
        {"name": "packed_100", "kind": "packed", "batch": 24, "heads": 16, "kv_heads": 4, "head_dim": 64, "rows": 100, "causal": True, "ragged": True},
        # a batch of an encoder's frames, each seeing all of its own
        {"name": "packed_1500", "kind": "packed", "batch": 4, "heads": 6, "kv_heads": 6, "head_dim": 64, "rows": 1500, "causal": False, "ragged": False},
        # one prompt, a head of keys for each of queries
        {"name": "packed_2048", "kind": "packed", "batch": 1, "heads": 24, "kv_heads": 24, "head_dim": 96, "rows": 2048, "causal": True, "ragged": False},
        # prompts of different lengths in one pass, four query heads on a head of keys: the most operations
        {"name": "packed_4096", "kind": "packed", "batch": 4, "heads": 32, "kv_heads": 8, "head_dim": 128, "rows": 4096, "causal": True, "ragged": True},
    ]


# what a drawn case may cost: the largest listed ones
MOST_BYTES, MOST_FLOPS = 6.9e8, 3.1e11


def draw(rng):
    def spread(lo, hi):
        return max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        kind = rng.choice(["write", "paged", "paged", "paged", "packed", "packed"])
        kv_heads = rng.choice([1, 2, 4, 6, 8, 16, 32])
        case = {"kind": kind, "batch": rng.choice([1, spread(1, 64), spread(1, 64)])}
        if kind != "write":
            case["heads"] = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
            if case["heads"] > 64:
                continue
        case.update({"kv_heads": kv_heads, "head_dim": rng.choice([64, 80, 96, 112, 128, 128])})
        if kind != "packed":
            case["page_size"] = rng.choice([16, 16, 32, 64, 128, 256])
        if kind == "write":
            case.update({"rows": rng.choice([1, spread(1, 4096)]), "before": rng.choice([0, spread(1, 4096)]), "source": rng.choice(["f16", "f16", "f32"])})
        elif kind == "paged":
            rows = rng.choice([1, 1, spread(2, 16), spread(2, 2048)])
            case.update({"rows": rows, "keys": rows + spread(16, 65536), "ragged": rng.random() < 0.7})
        else:
            case.update({"rows": spread(16, 8192), "causal": rng.random() < 0.8, "ragged": rng.random() < 0.7})
        # the plain forms hold the scores of every head, padded to the longest sequence, and a write's outputs are its pools
        if kind == "write" and case["batch"] * (case["rows"] + case["before"]) * kv_heads * case["head_dim"] > 6.0e7:
            continue
        if kind != "write" and case["batch"] * case["heads"] * case["rows"] * case.get("keys", case["rows"]) > 2.2e9:
            continue
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ---- inputs -------------------------------------------------------------------------------------------------------------


def counts(case):
    """Query rows of each sequence: a quarter of the longest to all of it, odd ones among them; one alike for a few."""
    b, rows = case["batch"], case["rows"]
    if rows <= 16 or not case.get("ragged", True):
        return [rows] * b
    return [max(1, rows - (i * rows * 3) // (4 * b)) for i in range(b)]


def lengths(case):
    """Keys of each sequence, its new rows among them."""
    n, b = counts(case), case["batch"]
    if case["kind"] == "packed":
        return n
    if case["kind"] == "write":
        return [case["before"] * (i % 3 + 1) // 3 + x for i, x in enumerate(n)]
    keys = case["keys"]
    return [max(x, keys - (i * keys * 3) // (4 * b)) if case["ragged"] else keys for i, x in enumerate(n)]


def rows_of(gen, shape):
    """Keys or values [..., heads, head_dim]: N(0, 1) with a spread and an offset of its own for each head's dimension, a few of them large."""
    one, two = (torch.randn(shape[-2:], generator=gen, device=GPU) for _ in range(2))
    return (torch.randn(shape, generator=gen, device=GPU) * torch.exp(0.4 * one) + 0.3 * two**3).half()


def starts_of(sizes):
    return torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32, device=GPU)


def prepare(case, seed):
    gen = torch.Generator(GPU)
    gen.manual_seed(seed)
    b, kv, d = case["batch"], case["kv_heads"], case["head_dim"]
    n, lens = counts(case), lengths(case)
    total = sum(n)
    state = {"case": case, "starts": starts_of(n)}
    if case["kind"] == "packed":
        h = case["heads"]
        q = torch.randn((total, h, d), generator=gen, device=GPU).half()
        # as a fused projection leaves them
        state["qkv"] = torch.cat([q, rows_of(gen, (total, kv, d)), rows_of(gen, (total, kv, d))], 1).view(total, (h + 2 * kv) * d)
        return state
    ps = case["page_size"]
    needs = [(x + ps - 1) // ps for x in lens]
    pages, width = sum(needs) + 3, max(needs) + 1
    # pages are given out in any order; where a sequence has none the table says -1
    order = torch.randperm(pages, generator=gen, device=GPU).to(torch.int32)
    at = starts_of(needs).long()
    j = torch.arange(width, device=GPU)
    state["table"] = torch.where(j < (at[1:] - at[:-1])[:, None], order[torch.clamp(at[:-1, None] + j, max=pages - 1)], -1).contiguous()
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device=GPU)
    for name in ("k_pool", "v_pool"):
        # (a head's rows are drawn alike, so that a pool's pages may go to any sequence)
        state[name] = rows_of(gen, (pages, ps, kv, d)).transpose(1, 2).contiguous()
    if case["kind"] == "write":
        state["k"], state["v"] = (rows_of(gen, (total, kv, d)).view(total, kv * d) for _ in range(2))
        if case["source"] == "f32":
            state["k"], state["v"] = (x.float() * (1 + 2.0**-12) for x in (state["k"], state["v"]))
    else:
        state["q"] = torch.randn((total, case["heads"] * d), generator=gen, device=GPU).half()
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------


def places(starts, total):
    """Sequence and row within it of every packed row."""
    r = torch.arange(total, device=GPU)
    b = torch.searchsorted(starts.long(), r, right=True) - 1
    return b, r - starts.long()[b]


def plain_write(state):
    case = state["case"]
    kv, d, ps, total = case["kv_heads"], case["head_dim"], case["page_size"], state["k"].shape[0]
    b, i = places(state["starts"], total)
    n = (state["starts"][1:] - state["starts"][:-1]).long()
    at = (state["lens"].long() - n)[b] + i
    page = state["table"].long()[b, at // ps]
    state["k_pool"][page, :, at % ps] = state["k"].half().view(total, kv, d)
    state["v_pool"][page, :, at % ps] = state["v"].half().view(total, kv, d)
    return [state["k_pool"], state["v_pool"]]


def plain_attention(q, k, v, n, lens, causal):
    """q [batch, rows, heads, d], k and v [batch, kv_heads, keys, d] in 32 bits, padded; n rows and lens keys of each -> [batch, rows, heads, d]."""
    b, rows, h, d = q.shape
    kv, keys = k.shape[1:3]
    g = h // kv
    q = q.view(b, rows, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * rows, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(d)).view(b, kv, g, rows, keys)
    last = (lens - 1)[:, None].expand(b, rows)
    if causal:
        last = torch.arange(rows, device=GPU)[None] + (lens - n)[:, None]
    s.masked_fill_((torch.arange(keys, device=GPU) > last[:, :, None])[:, None, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, kv, g * rows, keys), v).view(b, kv, g, rows, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(b, rows, h, d)


def plain_paged(state):
    case = state["case"]
    b, h, kv, d, ps = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim", "page_size"))
    total, rows, keys = state["q"].shape[0], max(counts(case)), max(lengths(case))
    pages = state["table"][:, : (keys + ps - 1) // ps].long().clamp(min=0)
    k, v = (state[x][pages].transpose(1, 2).reshape(b, kv, -1, d)[:, :, :keys].float() for x in ("k_pool", "v_pool"))
    starts, lens = state["starts"].long(), state["lens"].long()
    n = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + torch.arange(rows, device=GPU)).clamp(max=total - 1)
    # what lies behind a sequence's keys is another's: it is not seen, and its values are taken out
    v.masked_fill_((torch.arange(keys, device=GPU) >= lens[:, None])[:, None, :, None], 0)
    o = plain_attention(state["q"].view(total, h, d)[at].float(), k, v, n, lens, True)
    return o[places(state["starts"], total)].half().view(total, h * d)


def plain_packed(state):
    case = state["case"]
    h, kv, d = (case[x] for x in ("heads", "kv_heads", "head_dim"))
    total, rows = state["qkv"].shape[0], max(counts(case))
    starts = state["starts"].long()
    n = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + torch.arange(rows, device=GPU)).clamp(max=total - 1)
    x = state["qkv"].view(total, h + 2 * kv, d)[at].float()
    o = plain_attention(x[:, :, :h], x[:, :, h : h + kv].transpose(1, 2), x[:, :, h + kv :].transpose(1, 2).contiguous(), n, n, case["causal"])
    return o[places(state["starts"], total)].half().view(total, h * d)


# ---- the framework's calls --------------------------------------------------------------------------------------------------

_device = None


def library():
    """The library and its context: one for the program's life."""
    global _device
    import ratchet_amd as ra

    if _device is None:
        _device = ra.Device.request_device(ra.DeviceRequest.GPU)
    return ra.lib(), _device.ctx


def check(status):
    if status != 0:
        import ratchet_amd as ra

        L, ctx = library()
        raise RuntimeError(L.rt_last_error(ctx).decode() or ra._ffi.status_string(status))


class Compiled:
    """What a program makes once for these shapes and keeps: a descriptor, a workspace, the output; and the call."""

    def __init__(self, state):
        import ctypes

        from ratchet_amd import _ffi

        L, ctx = library()
        case, need = state["case"], ctypes.c_uint64()
        b, kv, d = case["batch"], case["kv_heads"], case["head_dim"]
        if case["kind"] != "packed":
            cache = _ffi.PagedCacheDesc()
            cache.batch, cache.kv_heads, cache.head_dim = b, kv, d
            cache.pages, cache.page_size = state["k_pool"].shape[0], case["page_size"]
            cache.table_width = cache.table_stride = state["table"].shape[1]
        if case["kind"] == "write":
            self.desc, self.out = cache, [state["k_pool"], state["v_pool"]]
            strides = (ctypes.c_int64 * 2)(kv * d, d)
            self.call = L.rt_cache_write_paged_enqueue
            self.args = (ctx, ctypes.byref(cache), _ffi.RT_F16 if case["source"] == "f16" else _ffi.RT_F32, state["k_pool"].data_ptr(), state["k"].data_ptr(),
                         state["v_pool"].data_ptr(), state["v"].data_ptr(), strides, state["table"].data_ptr(), state["lens"].data_ptr(), state["starts"].data_ptr(),
                         state["k"].shape[0])
            return
        h = case["heads"]
        if case["kind"] == "paged":
            desc = _ffi.AttentionPagedDesc()
            desc.cache, desc.rows = cache, state["q"].shape[0]
            desc.q_strides[:] = [h * d, d]
            size, desc.causal = L.rt_attention_paged_workspace_bytes, 1
            self.call = L.rt_attention_paged_enqueue
            args = (state["q"].data_ptr(), state["k_pool"].data_ptr(), state["v_pool"].data_ptr(), state["table"].data_ptr(), state["lens"].data_ptr(), state["starts"].data_ptr())
        else:
            desc = _ffi.AttentionPackedDesc()
            desc.batch, desc.kv_heads, desc.head_dim = b, kv, d
            desc.rows = desc.kv_rows = state["qkv"].shape[0]
            desc.q_strides[:] = desc.k_strides[:] = desc.v_strides[:] = [(h + 2 * kv) * d, d]
            size, desc.causal = L.rt_attention_packed_workspace_bytes, int(case["causal"])
            self.call = L.rt_attention_packed_enqueue
            at = state["qkv"].data_ptr()
            args = (at, at + 2 * h * d, at + 2 * (h + kv) * d, state["starts"].data_ptr(), None)
        desc.heads, desc.scale = h, 1 / math.sqrt(d)
        desc.max_rows, desc.max_keys = max(counts(case)), max(lengths(case))
        desc.o_strides[:] = [h * d, d]
        check(size(ctypes.byref(desc), ctypes.byref(need)))
        self.workspace = torch.empty(need.value, dtype=torch.uint8, device=GPU) if need.value else None
        self.out = torch.empty((desc.rows, h * d), dtype=torch.float16, device=GPU)
        self.desc, self.args = desc, (ctx, ctypes.byref(desc), *args, self.out.data_ptr(), self.workspace.data_ptr() if need.value else None, need.value)


def framework(state):
    made = state.get("compiled")
    if made is None:
        made = state["compiled"] = Compiled(state)
    check(made.call(*made.args, torch.cuda.current_stream().cuda_stream))
    return made.out


def run(state):
    if own:
        return framework(state)
    return {"write": plain_write, "paged": plain_paged, "packed": plain_packed}[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and the operators in 64 bits -------------------------------------------------------------


def work(case):
    kv, d, n, lens = case["kv_heads"], case["head_dim"], counts(case), lengths(case)
    if case["kind"] == "write":
        return {"bytes": 2.0 * sum(n) * kv * d * (2 + (4 if case["source"] == "f32" else 2)), "flops": 0.0}
    h = case["heads"]
    # (query, key) pairs of a head
    pairs = sum(x * (y - (x - 1) / 2 if case.get("causal", True) else y) for x, y in zip(n, lens))
    return {"bytes": 4.0 * d * (kv * sum(lens) + h * sum(n)), "flops": 4.0 * h * d * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    b, kv, d, n, lens = case["batch"], case["kv_heads"], case["head_dim"], counts(case), lengths(case)
    starts = [sum(n[:i]) for i in range(b + 1)]
    if case["kind"] != "packed":
        ps, table = case["page_size"], state["table"].tolist()
    if case["kind"] == "write":
        pools = [state["k_pool"].double(), state["v_pool"].double()]
        for i in range(b):
            at = lens[i] - n[i]
            while at < lens[i]:  # a page's rows at a time
                to = min(lens[i], (at // ps + 1) * ps)
                rows = slice(starts[i] + at - (lens[i] - n[i]), starts[i] + to - (lens[i] - n[i]))
                for pool, src in zip(pools, (state["k"], state["v"])):
                    pool[table[i][at // ps], :, at % ps : at % ps + to - at] = src[rows].double().view(-1, kv, d).transpose(0, 1)
                at = to
        return pools
    h = case["heads"]
    g, out = h // kv, torch.empty((starts[b], h, d), dtype=torch.float64, device=GPU)
    for i in range(b):
        rows, keys = slice(starts[i], starts[i + 1]), lens[i]
        if case["kind"] == "packed":
            x = state["qkv"][rows].view(-1, h + 2 * kv, d).double()
            q, k, v = x[:, :h], x[:, h : h + kv], x[:, h + kv :]
        else:
            pages = torch.tensor(table[i][: (keys + ps - 1) // ps], device=GPU)
            q = state["q"][rows].view(-1, h, d).double()
            k, v = (state[p][pages].permute(0, 2, 1, 3).reshape(-1, kv, d)[:keys].double() for p in ("k_pool", "v_pool"))
        hidden = torch.ones((n[i], keys), dtype=torch.bool, device=GPU).triu(keys - n[i] + 1) if case.get("causal", True) else None
        for head in range(h):
            s = q[:, head] @ k[:, head // g].T.contiguous() / math.sqrt(d)
            if hidden is not None:
                s.masked_fill_(hidden, float("-inf"))
            out[rows, head] = torch.softmax(s, -1) @ v[:, head // g].contiguous()
    return out.view(-1, h * d)
