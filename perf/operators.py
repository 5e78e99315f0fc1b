"""The operators on 4-bit blocks: products with Q4_0 weights, the write into a key/value cache held in 4 bits, and the attention that
reads such a cache.

Both forms of an operator take the same bytes.  A block is 32 consecutive values of a row with one f16 scale d and a 4-bit code q each,
value d * (q - 8); eight values are one dword whose nibbles 0..3 hold values 0, 2, 4, 6 and nibbles 4..7 values 1, 3, 5, 7.

  product    rows activation rows (1: a decode step of one sequence; a few: one step of several sequences; hundreds: a prompt) against an
             n x k weight, with bias, and with an activation behind it or none.  f16 activations.
  write      len new key and value rows of every sequence and head into their caches; the values as held come back.
             len = 1 is a decode step, more a prompt.
  attention  queries [batch, len, heads * head_dim] against a cache of kv_heads heads (heads / kv_heads queries share one).  rows = 1 is a
             decode step, a few are drafted tokens, many a prompt.  ragged: the sequences differ in length (a quarter of the longest to all
             of it); mask: none, the causal flag, or the mask as a tensor.

Shapes: the widths, head sizes and lengths of this repository's tests and benchmark (2560 x 10240 weights, 32 heads of 80 or 96, a vocabulary of 51865)
and generic ones around them; heads that share keys and values are usual where a cache is the bound.
"""
import math

import torch

own = False

GPU = "cuda:0"
ACTS = {"none": 0, "gelu": 1, "silu": 2}


def listed():
    return [
        # one token through an up-projection: latency and one pass over 15 MB
        {"name": "product_1", "kind": "product", "rows": 1, "n": 10240, "k": 2560, "act": "none"},
        # one step of four sequences through a down-projection: few weight rows, a long sum
        {"name": "product_4", "kind": "product", "rows": 4, "n": 2560, "k": 10240, "act": "none"},
        # sixteen sequences' logits over a vocabulary with an odd number of entries
        {"name": "product_16", "kind": "product", "rows": 16, "n": 51865, "k": 2560, "act": "none"},
        # a prompt through an up-projection with its activation
        {"name": "product_512", "kind": "product", "rows": 512, "n": 10240, "k": 2560, "act": "gelu"},
        # a decode step's new keys and values: latency
        {"name": "write_1", "kind": "write", "batch": 1, "heads": 32, "head_dim": 80, "rows": 1, "offset": 1023},
        # a batch of prompts
        {"name": "write_2048", "kind": "write", "batch": 4, "heads": 32, "head_dim": 96, "rows": 2048, "offset": 0},
        # a decode step with 1024 positions behind it, a head of keys for each of queries: latency
        {"name": "attention_1", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 32, "head_dim": 80, "rows": 1, "keys": 1024, "mask": "none",
         "ragged": False},
        # one long conversation, four query heads to a head of keys
        {"name": "attention_long", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "rows": 1, "keys": 32768, "mask": "none",
         "ragged": False},
        # a serving batch of sequences of different lengths: the most bytes
        {"name": "attention_batch", "kind": "attention", "batch": 32, "heads": 32, "kv_heads": 8, "head_dim": 128, "rows": 1, "keys": 8192, "mask": "none",
         "ragged": True},
        # drafted tokens of a few sequences
        {"name": "attention_7", "kind": "attention", "batch": 4, "heads": 32, "kv_heads": 32, "head_dim": 96, "rows": 7, "keys": 2001, "mask": "causal",
         "ragged": True},
        # the end of a prompt with its mask as a tensor
        {"name": "attention_150", "kind": "attention", "batch": 2, "heads": 16, "kv_heads": 4, "head_dim": 64, "rows": 150, "keys": 1373, "mask": "f16",
         "ragged": False},
        # a long prompt: the most operations
        {"name": "attention_2048", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 32, "head_dim": 96, "rows": 2048, "keys": 2048, "mask": "causal",
         "ragged": False},
    ]


# what a drawn case may cost: the largest listed ones
MOST_BYTES, MOST_FLOPS = 2.0e8, 2.6e10


def draw(rng):
    def spread(lo, hi, step=1):
        return max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step

    while True:
        kind = rng.choice(["product", "product", "write", "attention", "attention", "attention"])
        if kind == "product":
            case = {"kind": kind, "rows": rng.choice([1, spread(1, 16), spread(1, 512)]), "n": rng.choice([spread(256, 51865), spread(256, 16384, 32)]),
                    "k": rng.choice([spread(256, 12288, 256), spread(256, 12288, 32)]), "act": rng.choice(list(ACTS))}
        elif kind == "write":
            case = {"kind": kind, "batch": spread(1, 32), "heads": rng.choice([4, 6, 8, 16, 32]), "head_dim": rng.choice([64, 80, 96, 112, 128]),
                    "rows": rng.choice([1, spread(1, 4096)]), "offset": rng.choice([0, spread(1, 4096)])}
        else:
            kv_heads = rng.choice([1, 2, 4, 6, 8, 16, 32])
            rows = rng.choice([1, 1, spread(2, 16), spread(2, 2048)])
            case = {"kind": kind, "batch": rng.choice([1, spread(1, 64)]), "heads": kv_heads * rng.choice([1, 1, 2, 4, 5, 8]), "kv_heads": kv_heads,
                    "head_dim": rng.choice([64, 80, 96, 112, 128]), "rows": rows, "keys": rows + spread(16, 32768),
                    "mask": rng.choice(["none", "causal", "causal", "f16", "f32"]), "ragged": rng.random() < 0.5}
            if case["heads"] > 64 or case["mask"] in ("f16", "f32") and case["ragged"]:
                continue
            # the plain form holds the scores of every head at once
            if case["batch"] * case["heads"] * rows * case["keys"] > 1.4e8:
                continue
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ---- the format -------------------------------------------------------------------------------------------------------


def pad256(n):
    return (n + 255) // 256 * 256


def blocks_of(head_dim):
    return (head_dim + 31) // 32


def scales_of(head_dim):
    """Scales a cache row takes: its blocks', to the next of 1, 2, 4."""
    return 1 << (blocks_of(head_dim) - 1).bit_length()


def packed(q):
    """Codes 0..15 [..., D], D % 8 == 0 -> bytes [..., D / 2]."""
    n = q.to(torch.uint8).unflatten(-1, (-1, 4, 2)).transpose(-1, -2).flatten(-2)  # a dword's nibbles
    n = n.unflatten(-1, (4, 2))
    return (n[..., 0] | n[..., 1] << 4).flatten(-2)


def values(codes, scales, d):
    """Bytes [..., d / 2] and f16 scales [..., at least one for each 32 values] -> f32 values [..., d]."""
    n = torch.stack([codes & 15, codes >> 4], -1).unflatten(-2, (-1, 4)).flatten(-2)  # [..., dwords, 8 nibbles]
    q = n.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-3).float().sub_(8.0)
    return q.mul_(scales.float().repeat_interleave(32, -1)[..., :d])


def largest(x):
    """The value of largest magnitude along the last axis, the first of equals."""
    a = x.abs()
    at = torch.where(a == a.amax(-1, keepdim=True), torch.arange(x.shape[-1], device=x.device), x.shape[-1]).amin(-1, keepdim=True)
    return x.gather(-1, at).squeeze(-1)


def held(x):
    """f16 rows [..., D] as a cache holds them: codes [..., D] and f16 scales [..., blocks]."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -d % 32)).float().unflatten(-1, (-1, 32))
    m = largest(x)
    t = m.abs() / 8
    # eight significant bits, and nothing finer than 2^-24: every d * (q - 8) is an f16 number
    s = torch.where(t < 2.0**-17, t.half().float(), t.bfloat16().float()).clamp(max=8160.0)
    s = torch.where(m > 0, -s, s)
    # in 64 bits: a quotient half way between two codes has to come out as that
    q = torch.where(s[..., None] == 0, 8.0, torch.floor(x.double() / s[..., None].double() + 8.5)).clamp(0, 15)
    return q.flatten(-2)[..., :d], s.half()


def cache_of(x, capacity):
    """K or V rows [batch, heads, rows, D] as a cache of that capacity, its other rows zeros: one buffer of bytes."""
    b, h, rows, d = x.shape
    codes = torch.zeros((b, h, capacity, d // 2), dtype=torch.uint8, device=x.device)
    scales = torch.zeros((b, h, capacity, scales_of(d)), dtype=torch.float16, device=x.device)
    for i in range(b):  # (a sequence at a time: the quotients are in 64 bits)
        q, s = held(x[i])
        codes[i, :, :rows], scales[i, :, :rows, :blocks_of(d)] = packed(q), s
    return joined(codes, scales)


def joined(codes, scales):
    a, b = codes.reshape(-1), scales.reshape(-1).view(torch.uint8)
    out = torch.zeros(pad256(a.numel()) + pad256(b.numel()), dtype=torch.uint8, device=a.device)
    out[: a.numel()], out[pad256(a.numel()) : pad256(a.numel()) + b.numel()] = a, b
    return out


def parts(buf, lead, d, scales):
    """Views of a buffer's codes [*lead, d / 2] and scales [*lead, scales]."""
    rows = math.prod(lead)
    at = pad256(rows * d // 2)
    return buf[: rows * d // 2].view(*lead, d // 2), buf[at : at + 2 * rows * scales].view(torch.float16).view(*lead, scales)


# ---- inputs -------------------------------------------------------------------------------------------------------------


def lengths(case):
    b, keys = case["batch"], case["keys"]
    return [max(case["rows"], keys - i * keys * 3 // (4 * b)) if case["ragged"] else keys for i in range(b)]


def rows_of(gen, shape):
    """Keys or values: N(0, 1) with a spread and an offset of its own for each head's dimension, a few of them large."""
    one = torch.randn((1, shape[1], 1, shape[3]), generator=gen, device=GPU)
    two = torch.randn((1, shape[1], 1, shape[3]), generator=gen, device=GPU)
    return (torch.randn(shape, generator=gen, device=GPU) * torch.exp(0.4 * one) + 0.3 * two**3).half()


def prepare(case, seed):
    gen = torch.Generator(GPU)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=GPU)

    if case["kind"] == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        w = (normal(n, k) / math.sqrt(k)).view(-1, 32)
        d = (largest(w) / -8).half()
        q = torch.where(d[:, None] == 0, 8.0, torch.floor(w / d.float()[:, None] + 8.5)).clamp_(0, 15)
        return {"case": case, "w": joined(packed(q), d), "x": normal(rows, k).half(), "bias": (0.02 * normal(n)).half()}
    if case["kind"] == "write":
        b, h, d, rows, capacity = case["batch"], case["heads"], case["head_dim"], case["rows"], case["offset"] + case["rows"] + 3
        empty = joined(torch.zeros((b, h, capacity, d // 2), dtype=torch.uint8, device=GPU), torch.zeros((b, h, capacity, scales_of(d)), dtype=torch.float16, device=GPU))
        # as a projection leaves them: [batch, rows, heads * head_dim]
        k, v = (rows_of(gen, (b, h, rows, d)).transpose(1, 2).contiguous() for _ in range(2))
        return {"case": case, "k": k, "v": v, "k_cache": empty, "v_cache": empty.clone(), "capacity": capacity}
    b, h, kv, d, rows, keys = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim", "rows", "keys"))
    state = {"case": case, "q": normal(b, rows, h * d).half(), "mask": None, "lens": None, "capacity": keys + 5}
    for name in ("k_cache", "v_cache"):
        state[name] = cache_of(rows_of(gen, (b, kv, keys, d)), keys + 5)
    if case["ragged"]:
        state["lens"] = torch.tensor(lengths(case), dtype=torch.int32, device=GPU)
    if case["mask"] in ("f16", "f32"):  # 0 and -inf, as the callers make it
        hidden = torch.arange(keys, device=GPU)[None, :] > torch.arange(rows, device=GPU)[:, None] + (keys - rows)
        state["mask"] = torch.zeros((rows, keys), device=GPU).masked_fill_(hidden, float("-inf")).to(torch.float16 if case["mask"] == "f16" else torch.float32)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------


def activation(y, act):
    # gelu: x * (0.5 + 0.5 * tanh(u)) with u = x * (0.035677407 x^2 + 0.7978846); silu: x * sigmoid(x)
    if act == "none":
        return y
    z = y if act == "silu" else 2 * y * (0.035677407 * y * y + 0.7978846)
    return y / (1 + torch.exp(-z))


def plain_product(state):
    case = state["case"]
    codes, scales = parts(state["w"], (case["n"], case["k"] // 32), 32, 1)
    w = values(codes, scales, 32).view(case["n"], case["k"])
    return activation(torch.matmul(state["x"].float(), w.t()) + state["bias"].float(), case["act"]).half()


def plain_write(state):
    case = state["case"]
    b, h, d, rows, at = (case[x] for x in ("batch", "heads", "head_dim", "rows", "offset"))
    out = []
    for new, cache in ((state["k"], state["k_cache"]), (state["v"], state["v_cache"])):
        q, s = held(new.view(b, rows, h, d).transpose(1, 2))
        codes, scales = parts(cache, (b, h, state["capacity"]), d, scales_of(d))
        p = packed(q)
        codes[:, :, at : at + rows], scales[:, :, at : at + rows, : blocks_of(d)] = p, s
        out.append(values(p, s, d).half())
    return out


def plain_attention(state):
    case = state["case"]
    b, h, kv, d, rows, keys = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim", "rows", "keys"))
    g = h // kv
    codes, scales = parts(state["k_cache"], (b, kv, state["capacity"]), d, scales_of(d))
    k = values(codes[:, :, :keys], scales[:, :, :keys], d)
    codes, scales = parts(state["v_cache"], (b, kv, state["capacity"]), d, scales_of(d))
    v = values(codes[:, :, :keys], scales[:, :, :keys], d)
    q = state["q"].float().view(b, rows, kv, g, d).permute(0, 2, 4, 3, 1).reshape(b, kv, d, g * rows)
    s = torch.matmul(k, q).transpose(-1, -2).contiguous().mul_(1 / math.sqrt(d)).view(b, kv, g, rows, keys)
    if state["mask"] is not None:
        s = s + state["mask"].float()
    lens = torch.full((b,), keys, device=GPU) if state["lens"] is None else state["lens"]
    j = torch.arange(keys, device=GPU)
    last = (lens - 1)[:, None] if case["mask"] != "causal" else torch.arange(rows, device=GPU)[None, :] + (lens - rows)[:, None]
    if case["mask"] == "causal" or state["lens"] is not None:
        s = s.masked_fill_((j[None, None, :] > last[:, :, None])[:, None, None], float("-inf"))
    s = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul((s / s.sum(-1, keepdim=True)).view(b, kv, g * rows, keys), v)
    return o.view(b, kv, g, rows, d).permute(0, 3, 1, 2, 4).reshape(b, rows, h * d).half()


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
    """What a program makes once for these shapes and keeps: a descriptor or plan, a workspace, outputs; and the call."""

    def __init__(self, state):
        import ctypes

        from ratchet_amd import _ffi

        L, ctx = library()
        case, need, ws = state["case"], ctypes.c_uint64(), None
        self.plan = None
        if case["kind"] == "product":
            rows, n, k = case["rows"], case["n"], case["k"]
            # the reference's Linear: W.gemm(x, bias, false, true, true)
            desc = _ffi.make_desc(_ffi.RT_Q4_0, (n, k), _ffi.RT_F16, (rows, k), False, True, True, _ffi.RT_F16, (n,))
            self.plan, self.destroy = ctypes.c_void_p(), L.rt_matmul_plan_destroy
            check(L.rt_matmul_plan_create(ctx, ctypes.byref(desc), ACTS[case["act"]], ctypes.byref(self.plan)))
            check(L.rt_matmul_workspace_bytes(ctx, ctypes.byref(desc), ctypes.byref(need)))
            ws = torch.empty(need.value, dtype=torch.uint8, device=GPU) if need.value else None
            self.out = torch.empty((rows, n), dtype=torch.float16, device=GPU)
            self.call, self.args = L.rt_matmul_plan_enqueue, (self.plan, state["w"].data_ptr(), state["x"].data_ptr(), state["bias"].data_ptr(), self.out.data_ptr(),
                                                              ws.data_ptr() if need.value else None, need.value)
        elif case["kind"] == "write":
            b, h, d, rows = (case[x] for x in ("batch", "heads", "head_dim", "rows"))
            self.out = [torch.empty((b, h, rows, d), dtype=torch.float16, device=GPU) for _ in range(2)]
            strides = (ctypes.c_int64 * 3)(rows * h * d, d, h * d)
            self.call, self.args = L.rt_cache_write_q4_enqueue, (ctx, _ffi.RT_F16, state["k_cache"].data_ptr(), state["k"].data_ptr(), state["v_cache"].data_ptr(),
                                                                 state["v"].data_ptr(), strides, self.out[0].data_ptr(), self.out[1].data_ptr(), None, b, h,
                                                                 state["capacity"], case["offset"], rows, d)
        else:
            b, h, d, rows = (case[x] for x in ("batch", "heads", "head_dim", "rows"))
            desc = _ffi.AttentionQ4Desc()
            desc.batch, desc.heads, desc.kv_heads, desc.q_len, desc.kv_len, desc.head_dim, desc.capacity = b, h, case["kv_heads"], rows, case["keys"], d, state["capacity"]
            desc.q_strides[:] = desc.o_strides[:] = [rows * h * d, d, h * d]
            desc.scale, desc.causal = 1 / math.sqrt(d), int(case["mask"] == "causal")
            desc.mask_dtype = _ffi.RT_F16 if case["mask"] == "f16" else _ffi.RT_F32
            desc.mask_strides[:] = [0, case["keys"]]
            check(L.rt_attention_q4_workspace_bytes(ctypes.byref(desc), ctypes.byref(need)))
            ws = torch.empty(need.value, dtype=torch.uint8, device=GPU) if need.value else None
            self.out = torch.empty_like(state["q"])
            self.call, self.args = L.rt_attention_q4_enqueue, (ctx, ctypes.byref(desc), state["q"].data_ptr(), state["k_cache"].data_ptr(), state["v_cache"].data_ptr(),
                                                               None if state["mask"] is None else state["mask"].data_ptr(),
                                                               None if state["lens"] is None else state["lens"].data_ptr(), self.out.data_ptr(),
                                                               ws.data_ptr() if need.value else None, need.value)
            self.desc = desc
        self.workspace = ws

    def __del__(self):
        if self.plan is not None:
            self.destroy(self.plan)


def framework(state):
    made = state.get("compiled")
    if made is None:
        made = state["compiled"] = Compiled(state)
    check(made.call(*made.args, torch.cuda.current_stream().cuda_stream))
    return made.out


def run(state):
    if own:
        return framework(state)
    return {"product": plain_product, "write": plain_write, "attention": plain_attention}[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and the operators in 64 bits -------------------------------------------------------------


def work(case):
    if case["kind"] == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k * (0.5 + 2 / 32) + 2.0 * (rows * k + n + rows * n), "flops": 2.0 * rows * n * k}
    d = case["head_dim"]
    row = d / 2 + 2 * blocks_of(d)  # bytes of a cached row: codes and scales
    if case["kind"] == "write":
        rows = 2.0 * case["batch"] * case["heads"] * case["rows"]
        return {"bytes": rows * (2 * d + row + 2 * d), "flops": rows * d * 4}
    b, h, rows, lens = case["batch"], case["heads"], case["rows"], lengths(case)
    seen = sum(n - (rows - 1) / 2 if case["mask"] != "none" else n for n in lens)  # keys a query sees, on average, over the batch
    mask = rows * case["keys"] * {"f16": 2, "f32": 4}.get(case["mask"], 0)
    return {"bytes": 2.0 * case["kv_heads"] * sum(lens) * row + 4.0 * b * rows * h * d + mask, "flops": 4.0 * h * d * rows * seen}


def exact_values(buf, lead, d, scales, last=None):
    """Values in 64 bits from a buffer's dwords: value e of eight is nibble e / 2 of the low half (even e) or of the high half (odd e)."""
    count = math.prod(lead)
    words = buf[: count * d // 2].view(torch.int32).view(*lead, d // 8)
    at = pad256(count * d // 2)
    s = buf[at : at + 2 * count * scales].view(torch.float16).view(*lead, scales)
    if last is not None:
        words, s = words[..., :last, :], s[..., :last, :]
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=buf.device)
    q = (words[..., None] >> shift) & 15
    block = torch.arange(d, device=buf.device) // 32
    return (q.flatten(-2).double() - 8) * s.double()[..., block]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "product":
        w = exact_values(state["w"], (case["n"], case["k"] // 32), 32, 1).view(case["n"], case["k"])
        y = state["x"].double() @ w.T + state["bias"].double()
        if case["act"] == "gelu":
            return y * (0.5 + 0.5 * torch.tanh(y * (0.035677407 * y**2 + 0.7978846)))
        return y * torch.sigmoid(y) if case["act"] == "silu" else y
    b, d, rows = case["batch"], case["head_dim"], case["rows"]
    if case["kind"] == "write":
        out = []
        for x in (state["k"], state["v"]):
            x = x.view(b, rows, case["heads"], d).permute(0, 2, 1, 3).double()
            y = torch.empty_like(x)
            for lo in range(0, d, 32):
                z = x[..., lo : lo + 32]
                hi, low = z.amax(-1), z.amin(-1)
                first_hi = torch.where(z == hi[..., None], torch.arange(z.shape[-1], device=GPU), 99).amin(-1)
                first_low = torch.where(z == low[..., None], torch.arange(z.shape[-1], device=GPU), 99).amin(-1)
                m = torch.where((hi > -low) | ((hi == -low) & (first_hi < first_low)), hi, low)
                e = torch.frexp(m.abs() / 8)[1].long()  # |m| / 8 in [2^(e - 1), 2^e)
                unit = (torch.clamp(e - 8, min=-24) + 1023 << 52).view(torch.float64)  # 2^(e - 8): a power function may be an ulp off
                s = torch.clamp(torch.round(m.abs() / 8 / unit) * unit, max=8160.0) * -torch.sign(m)
                q = torch.floor(z / torch.where(s == 0, 1.0, s)[..., None] + 8.5).clamp(0, 15)
                y[..., lo : lo + 32] = (q - 8) * s[..., None]
            out.append(y)
        return out
    h, kv, keys = case["heads"], case["kv_heads"], case["keys"]
    g, lead = h // kv, (b, kv, state["capacity"])
    out = torch.empty((b, rows, h, d), dtype=torch.float64, device=GPU)
    k, v = (exact_values(state[x], lead, d, scales_of(d), keys) for x in ("k_cache", "v_cache"))
    for i, n in enumerate(lengths(case)):
        q = state["q"][i].double().view(rows, kv, g, d)
        for head in range(kv):
            s = (q[:, head].reshape(rows * g, d) @ k[i, head, :n].T.contiguous()).view(rows, g, n) / math.sqrt(d)
            if state["mask"] is not None:
                s = s + state["mask"][:, None, :n].double()
            if case["mask"] == "causal":
                s = s + torch.full((rows, n), float("-inf"), dtype=torch.float64, device=GPU).triu(n - rows + 1)[:, None, :]
            out[i, :, head * g : (head + 1) * g] = (torch.softmax(s, -1).view(rows * g, n) @ v[i, head, :n]).view(rows, g, d)
    return out.view(b, rows, h * d)
