"""The operators of the paged MX key/value cache as cases with inputs, a plain form in elementary torch operations, and
the calls a user makes of this package: writing keys and values into the pages (`paged_kv_append`), reading them back as
dense tensors (`paged_kv_gather`), the attention of one new token per sequence over the pages (`paged_attention`, with or
without the accumulated weight of every cached token) and the eviction of the tokens with the least accumulated weight
(`paged_kv_evict`).

A cache holds, for every page, key/value head and slot, one row of head_dim elements:
    none  bf16 values                                                       [pages, heads, slots, dim]
    mxfp  codes sign | exponent | fraction, one per byte (E4M3, E5M2) or two per byte (E2M1, element 2i in the low
          nibble), and one E8M0 byte per 32 elements                        [pages, heads, slots, dim / 32]
    mxint mantissas as int8 (in uint8 storage) and one biased exponent byte per 32 elements
Sequence b's token i lives in slot i % slots of page page_table[b, i // slots]; entries behind the last page are -1.
"""

import math
import random

import torch

own = False

FORMATS = {  # name -> (kind, exponent bits, fraction bits) or ("mxint", bits, 0)
    "none": ("none", 0, 0),
    "e4m3": ("mxfp", 4, 3),
    "e5m2": ("mxfp", 5, 2),
    "e2m1": ("mxfp", 2, 1),
    "int8": ("mxint", 8, 0),
}
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEVICE = "cuda"


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def _case(op, batch, heads, kv_heads, dim, page, low, high, fmt, dtype="bf16", **more):
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "low": low,
            "high": high, "fmt": fmt, "dtype": dtype, **more}


def listed():
    return [
        # one user at the start of a conversation: the latency of the smallest call
        {"name": "decode one short", **_case("decode", 1, 32, 8, 128, 16, 257, 257, "e4m3")},
        # a serving batch in mid-flight: 32 sequences of 1 to 8192 cached tokens
        {"name": "decode batch", **_case("decode", 32, 32, 8, 128, 64, 1, 8192, "e4m3")},
        # two very long documents: few rows, so the length has to be split over the GPU
        {"name": "decode long", **_case("decode", 2, 32, 8, 128, 64, 100001, 131072, "int8")},
        # a model without grouped heads and an unquantized cache, odd lengths
        {"name": "decode plain cache", **_case("decode", 16, 32, 32, 64, 32, 777, 2049, "none")},
        # the narrowest cache: many sequences, 64 query heads over 8, MXFP4 pages
        {"name": "decode fp4", **_case("decode", 64, 64, 8, 128, 64, 500, 4096, "e2m1")},
        # fp32 activations over E5M2 pages, one key/value head per query head, an empty sequence among them
        {"name": "decode fp32", **_case("decode", 5, 12, 12, 64, 16, 0, 1531, "e5m2", "fp32")},
        # decoding with the accumulated weight of every cached token kept for a later eviction
        {"name": "decode tracked", **_case("tracked", 8, 32, 8, 128, 64, 3000, 8192, "e4m3")},
        # one decoding step of a small batch: the new token's key and value go into the cache, then it attends
        {"name": "step", **_case("step", 16, 32, 8, 128, 16, 100, 1023, "int8")},
        # a prompt chunk: its keys and values go into the cache and the chunk's attention reads all that is cached
        {"name": "prompt", **_case("prompt", 4, 32, 8, 128, 64, 0, 512, "e4m3", tokens=2048)},
        # short ragged prompts of an fp32 model behind odd prefixes, MXFP4 pages
        {"name": "prompt ragged", **_case("prompt", 3, 8, 4, 64, 16, 5, 130, "e2m1", "fp32", tokens=211)},
        # one sequence over its budget
        {"name": "evict one", **_case("evict", 1, 32, 8, 128, 16, 1500, 1500, "none", keep=1024, recent=128)},
        # a batch of long sequences halved
        {"name": "evict batch", **_case("evict", 8, 32, 8, 128, 64, 12000, 16384, "none", keep=8192, recent=512)},
    ]


def _log_int(rng, low, high):
    return min(high, int(low * math.exp(rng.random() * math.log((high + 0.999) / low))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "tracked", "step", "prompt", "evict"])
    dim = rng.choice([32, 64, 64, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    fmt = rng.choice(["none", "e4m3", "e4m3", "e5m2", "e2m1", "int8", "int8"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    batch = _log_int(rng, 1, 48)
    most = 150_000_000 if op in ("decode", "tracked", "step") else 50_000_000  # elements of one side of the cache
    room = max(8, most // (batch * kv_heads * dim))
    high = _log_int(rng, 1, min(room, 100_000))
    low = rng.choice([0, 1, high // 2, high])
    if op == "prompt":
        tokens = _log_int(rng, 1, min(room, 4096))
        return _case(op, batch, kv_heads * group, kv_heads, dim, page, low % 700, min(high, 700), fmt, dtype, tokens=tokens)
    if op == "evict":  # pages of 16-bit values: moved rows are compared as they are
        high = max(high, 40)
        keep = rng.randint(20, high)
        return _case(op, batch, kv_heads * group, kv_heads, dim, page, high // 2, high, "none", dtype, keep=keep,
                     recent=rng.randint(0, keep))
    return _case(op, batch, kv_heads * group, kv_heads, dim, page, low, high, fmt, dtype)


def _lengths(case):
    """Cached tokens per sequence before the pass: the first has `high`, the last `low`, the rest spread between."""
    n, low, high = case["batch"], min(case["low"], case["high"]), case["high"]
    got = [low + (high - low) * ((i * 2654435761 + 97) % 4294967296) // 4294967296 for i in range(n)]
    got[-1], got[0] = low, high
    return got


def _counts(case):
    """Tokens per sequence of a prompt chunk: the first has all, the others up to a quarter fewer."""
    t = case["tokens"]
    return [t - (t // 4) * ((i * 40503) % 65536) // 65536 for i in range(case["batch"])]


def work(case):
    kind, e, f = FORMATS[case["fmt"]]
    bits = {"none": 16.0, "mxfp": 8.25 if e + f > 3 else 4.25, "mxint": 8.25}[kind]
    row = case["dim"] * bits / 8  # bytes of one key or value row in the pages
    dense = case["dim"] * (2 if case["dtype"] == "bf16" else 4)
    lens = _lengths(case)
    hkv, hq, n = case["kv_heads"], case["heads"], case["batch"]
    if case["op"] in ("decode", "tracked", "step"):
        total = sum(lens) + (n if case["op"] == "step" else 0)
        b = 2 * total * hkv * row + 2 * n * hq * dense
        if case["op"] == "tracked":
            b += 8 * total * hkv
        if case["op"] == "step":
            b += 2 * n * hkv * (dense + row)
        return {"bytes": b, "flops": 4.0 * total * hq * case["dim"]}
    if case["op"] == "prompt":
        new = sum(_counts(case))
        total = sum(lens) + new
        out = n * hkv * max(a + c for a, c in zip(lens, _counts(case)))  # rows behind a sequence's last are zeros
        return {"bytes": 2 * new * hkv * (dense + row) + 2 * total * hkv * row + 2 * out * dense,
                "flops": 2.0 * new * hkv * case["dim"] * 4}
    moved = sum(_expected_moves(x, case) for x in lens) * hkv
    stats = n * hkv * _width(case) * 8.0 * 2  # weights and positions, read and written
    return {"bytes": stats + 2 * 2 * moved * row, "flops": 4.0 * sum(lens) * hkv}


def _width(case):
    return -(-max(_lengths(case)) // case["page"]) * case["page"]


def _expected_moves(length, case):
    """Rows that change their slot: every protected token and every other kept one that sits behind the budget."""
    keep, recent = case["keep"], case["recent"]
    if length <= keep:
        return 0
    rest, left = keep - recent, length - recent
    return recent * min(1.0, (length - keep) / max(1, recent)) + rest * max(0, left - keep) / max(1, left)


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    op, n, hkv, hq, dim, page = (case[k] for k in ("op", "batch", "kv_heads", "heads", "dim", "page"))
    dtype = DTYPES[case["dtype"]]
    lens = _lengths(case)
    new = _counts(case) if op == "prompt" else [1] * n if op == "step" else [0] * n
    after = [a + b for a, b in zip(lens, new)]
    need = [-(-x // page) for x in after]
    width = max(1, max(need))
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    table = torch.full((n, width), -1, dtype=torch.int32)
    for i, k in enumerate(need):
        table[i, :k] = torch.tensor([order.pop() for _ in range(k)], dtype=torch.int32)

    # keys have a few channels of larger magnitude, as rotary keys of language models do; values are plainer
    channels = torch.exp(0.6 * torch.randn(hkv, 1, dim, generator=g, device=DEVICE))

    def rows(*shape):
        return torch.randn(*shape, dim, generator=g, device=DEVICE)

    state = {"case": dict(case), "table": table.to(DEVICE), "scaling": dim ** -0.5, "most": max(after)}
    for side in ("key", "value"):
        codes, scales = [], []
        for at in range(0, pages, 256):  # in pieces: the whole cache in fp32 would be large
            x = rows(min(256, pages - at), hkv, page).mul_(channels if side == "key" else 0.8).to(torch.bfloat16)
            c, s = _encode(x, case["fmt"])
            codes.append(c)
            scales.append(s)
        state[side + "_pages"] = torch.cat(codes)
        state[side + "_scales"] = torch.cat(scales) if scales[0] is not None else None
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    state["lengths"], state["after"] = as_int(lens), as_int(after)
    if op in ("decode", "tracked", "step"):
        state["query"] = (rows(n, hq, 1) * 1.2).to(dtype)
    if op == "tracked":  # what earlier steps left: most tokens near nothing, a few heavy
        state["weights"] = torch.exp(2 * torch.randn(n, hkv, width * page, generator=g, device=DEVICE) - 6)
    if op in ("prompt", "step"):
        t = case["tokens"] if op == "prompt" else 1
        # as a projection leaves them: [batch, tokens, heads, dim], seen as [batch, heads, tokens, dim]
        state["key"] = (rows(n, t, hkv) * channels.transpose(0, 1)).to(dtype).transpose(1, 2)
        state["value"] = (rows(n, t, hkv) * 0.8).to(dtype).transpose(1, 2)
        state["counts"] = as_int(new)
    if op == "evict":
        w = torch.exp(2 * torch.randn(n, hkv, width * page, generator=g, device=DEVICE) - 4)
        live = torch.arange(width * page, device=DEVICE) < state["lengths"][:, None, None]
        state["weights"] = torch.where(live, w, torch.zeros_like(w))
        # earlier evictions have left the tokens in no order of age
        shuffle = torch.rand(n, hkv, width * page, generator=g, device=DEVICE).masked_fill(~live, 2.0).argsort(-1)
        ages = torch.argsort(shuffle, -1).to(torch.int32)
        state["positions"] = torch.where(live, ages, torch.full_like(ages, -1))
    return state


# ----------------------------------------------------------------------------------------------------------------------
# plain forms of the formats
# ----------------------------------------------------------------------------------------------------------------------
def _encode(x, fmt):
    """Codes and shared exponents of x[..., dim] in blocks of 32 elements (bf16 values for the unquantized cache)."""
    kind, e, f = FORMATS[fmt]
    if kind == "none":
        return x.to(torch.bfloat16), None
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    wide = blocks.float()
    if kind == "mxint":
        top = blocks.abs().amax(-1, keepdim=True).clamp(min=torch.finfo(x.dtype).tiny)
        s = torch.log2(top).ceil().float()  # in the tensor's own type
        mant = torch.round(wide * torch.exp2(-s) * 2.0 ** (e - 1)).clamp(-(2.0 ** (e - 1)), 2.0 ** (e - 1) - 1)
        return (mant.to(torch.int8).view(torch.uint8).reshape(x.shape),
                (s + 127).clamp(0, 255).to(torch.uint8).squeeze(-1))
    bits = wide.view(torch.int32)
    mag = bits & 0x7FFFFFFF
    exp = mag >> 23
    top = torch.where(exp == 0, 0, mag).amax(-1, keepdim=True)
    bias, last = 2 ** (e - 1) - 1, 2 ** e - 1
    shared = torch.where(top == 0, -127, ((top >> 23) - 127 - (last - bias)).clamp(-127, 128))
    ye = exp - (127 + shared - bias)
    m15 = (mag >> 8) & 0x7FFF  # the low 8 mantissa bits are dropped before rounding
    cut = 15 - f
    frac = (m15 + ((1 << (cut - 1)) - 1) + ((m15 >> cut) & 1)) >> cut  # half to even
    frac = torch.where((ye == 0) & (frac != 0), (frac | (1 << f)) >> 1, frac)  # one truncating subnormal binade
    gone, over = (ye < 0) | (exp == 0), ye > last
    frac = torch.where(gone, 0, torch.where(over, (1 << f) - 1, frac))
    ye = torch.where(gone, 0, ye.clamp(max=last))
    lost = (exp - 127 - shared < -150) | ((exp - 127 - shared == -150) & ((mag & 0x7FFFFF) == 0))
    sign = (bits < 0) & (exp != 0) & ~lost
    code = ((ye << f) | frac) | torch.where(sign, 1 << (e + f), 0)
    code = code.reshape(x.shape).to(torch.uint8)
    if e + f == 3:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code, (shared + 127).to(torch.uint8).squeeze(-1)


def _table(fmt):
    """The value of every code in units of the block's scale, fp32 [256] (or [16])."""
    kind, e, f = FORMATS[fmt]
    code = torch.arange(16 if e + f == 3 else 256, device=DEVICE, dtype=torch.int32)
    if kind == "mxint":
        return torch.where(code > 127, code - 256, code).float() * 2.0 ** (1 - e)
    bias = 2 ** (e - 1) - 1
    ye, frac = (code >> f) & (2 ** e - 1), (code & (2 ** f - 1)).float()
    mag = torch.where(ye == 0, frac * 2.0 ** (1 - bias - f), (1 + frac * 2.0 ** -f) * torch.exp2((ye - bias).float()))
    return torch.where((code >> (e + f)) & 1 == 1, -mag, mag)


def _decode(codes, scales, fmt):
    """fp32 values of code rows [..., row bytes] with scales [..., dim / 32]."""
    if fmt == "none":
        return codes.float()
    if FORMATS[fmt][1] + FORMATS[fmt][2] == 3:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = _table(fmt)[codes.int()]
    s = torch.exp2(scales.float() - 127)
    return (v.view(*v.shape[:-1], -1, 32) * s.unsqueeze(-1)).flatten(-2)


def _read(state, side, tokens):
    """fp32 [batch, kv_heads, tokens, dim] of the cached rows (rows behind a sequence's last are whatever was read)."""
    case, page = state["case"], state["case"]["page"]
    cols = -(-tokens // page)
    table = state["table"][:, :cols].clamp(min=0).long()

    def dense(pages):  # [batch, cols, heads, page, row] -> [batch, heads, tokens, row]
        x = pages[table].transpose(1, 2)
        return x.reshape(*x.shape[:2], cols * page, x.shape[-1])[:, :, :tokens]

    codes = dense(state[side + "_pages"])
    scales = state[side + "_scales"]
    return _decode(codes, None if scales is None else dense(scales), case["fmt"])


# ----------------------------------------------------------------------------------------------------------------------
# plain forms of the operators
# ----------------------------------------------------------------------------------------------------------------------
def _plain_append(state):
    case = state["case"]
    page, t = case["page"], state["key"].shape[2]
    step = torch.arange(t, device=DEVICE)
    slot = state["lengths"][:, None].long() + step
    seq, tok = torch.nonzero(step[None, :] < state["counts"][:, None], as_tuple=True)
    at = slot[seq, tok]
    where = state["table"][seq, at // page].long()
    for side in ("key", "value"):
        codes, scales = _encode(state[side].contiguous(), case["fmt"])
        state[side + "_pages"][where, :, at % page] = codes[seq, :, tok]
        if scales is not None:
            state[side + "_scales"][where, :, at % page] = scales[seq, :, tok]


def _plain_gather(state, lengths, most):
    dtype = DTYPES[state["case"]["dtype"]]
    live = (torch.arange(most, device=DEVICE) < lengths[:, None])[:, None, :, None]
    return [torch.where(live, _read(state, side, most), 0.0).to(dtype) for side in ("key", "value")]


def _plain_attention(state, lengths, most, weights=None):
    case = state["case"]
    n, hkv, g, dim = case["batch"], case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    if most == 0:
        return torch.zeros_like(state["query"])
    live = (torch.arange(most, device=DEVICE) < lengths[:, None])[:, None, None, :]
    q = state["query"].float().view(n, hkv, g, dim)
    s = torch.where(live, torch.matmul(q, _read(state, "key", most).transpose(2, 3)) * state["scaling"], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(live, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = torch.where(live.transpose(2, 3), _read(state, "value", most), 0.0)
    if weights is not None:
        weights[:, :, :most] += p.sum(2)
    return torch.matmul(p, v).view(n, hkv * g, 1, dim).to(state["query"].dtype)


def _plain_evict(state):
    case = state["case"]
    keep, recent, page = case["keep"], case["recent"], case["page"]
    weights, positions, lens = state["weights"], state["positions"], state["lengths"][:, None, None]
    width = weights.shape[-1]
    at = torch.arange(width, device=DEVICE).expand_as(weights)
    live = at < lens
    key = torch.where(positions >= lens - recent, math.inf, weights)
    key = torch.where(live, key, -math.inf)
    rank = torch.argsort(torch.sort(key, dim=-1, descending=True, stable=True).indices, -1)
    kept = live & (rank < keep)
    new_len = torch.minimum(lens, torch.full_like(lens, keep))
    hole, mover = (at < new_len) & ~kept, (at >= new_len) & kept
    # the i-th hole takes the i-th mover
    order_hole = torch.sort(hole.to(torch.int8), dim=-1, descending=True, stable=True).indices
    order_mover = torch.sort(mover.to(torch.int8), dim=-1, descending=True, stable=True).indices
    used = at < hole.sum(-1, keepdim=True)
    b, h, i = torch.nonzero(used, as_tuple=True)
    dst, src = order_hole[b, h, i], order_mover[b, h, i]
    page_of = lambda slot: state["table"][b, slot // page].long()  # noqa: E731
    for pages in (state["key_pages"], state["value_pages"], state["key_scales"], state["value_scales"]):
        if pages is not None:
            pages[page_of(dst), h, dst % page] = pages[page_of(src), h, src % page]
    out_w, out_p = weights.clone(), positions.clone()
    out_w[b, h, dst], out_p[b, h, dst] = weights[b, h, src], positions[b, h, src]
    behind = at >= new_len
    return (new_len.view(-1), torch.where(behind, 0.0, out_w), torch.where(behind, -1, out_p),
            state["key_pages"], state["value_pages"])


def _cache(state):
    """The package's handle on the pages, made at the first pass on a state and kept, as a program keeps it."""
    if "cache" not in state:
        import mase_b200 as mb

        kind, e, f = FORMATS[state["case"]["fmt"]]
        config = {"mxfp": {"data_in_block_size": 32, "data_in_exponent_width": e, "data_in_frac_width": f},
                  "mxint": {"data_in_block_size": 32, "data_in_width": e}}.get(kind)
        state["cache"] = mb.PagedKVCache.from_pages(state["key_pages"], state["value_pages"], state["key_scales"],
                                                    state["value_scales"], None if kind == "none" else kind, config)
    return state["cache"]


def run(state):
    op = state["case"]["op"]
    if own:
        import mase_b200 as mb

        cache, table, lens = _cache(state), state["table"], state["lengths"]
        if op == "decode":
            return mb.paged_attention(cache, state["query"], table, lens, state["scaling"])
        if op == "tracked":
            return mb.paged_attention(cache, state["query"], table, lens, state["scaling"],
                                      weights=state["weights"]), state["weights"]
        if op == "step":
            mb.paged_kv_append(cache, state["key"], state["value"], table, lens)
            return mb.paged_attention(cache, state["query"], table, state["after"], state["scaling"])
        if op == "prompt":
            mb.paged_kv_append(cache, state["key"], state["value"], table, lens, counts=state["counts"])
            return mb.paged_kv_gather(cache, table, state["after"], state["most"], state["key"].dtype)
        c = state["case"]
        lens, weights, positions = mb.paged_kv_evict(cache, table, lens, state["weights"], c["keep"], c["recent"],
                                                     positions=state["positions"], next_position=lens)
        return lens, weights, positions, state["key_pages"], state["value_pages"]
    if op == "decode":
        return _plain_attention(state, state["lengths"], state["most"])
    if op == "tracked":
        return _plain_attention(state, state["lengths"], state["most"], state["weights"]), state["weights"]
    if op == "step":
        _plain_append(state)
        return _plain_attention(state, state["after"], state["most"])
    if op == "prompt":
        _plain_append(state)
        return _plain_gather(state, state["after"], state["most"])
    return _plain_evict(state)


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ----------------------------------------------------------------------------------------------------------------------
def _value_of(code, fmt):
    """float64 values of codes held one per element, by arithmetic on the code's fields."""
    kind, e, f = FORMATS[fmt]
    c = code.to(torch.int64)
    if kind == "mxint":
        return ((c ^ 128) - 128).double() / 2 ** (e - 1)
    field, frac, bias = (c >> f) % 2 ** e, c % 2 ** f, 2 ** (e - 1) - 1
    v = torch.ldexp((frac + torch.where(field > 0, 2 ** f, 0)).double(), field.clamp(min=1) - bias - f)
    return v * (1 - 2 * (c >> (e + f))).double()


def _exact_rows(state, side, b, length):
    case = state["case"]
    hkv, dim, page, fmt = case["kv_heads"], case["dim"], case["page"], case["fmt"]
    if length == 0:
        return torch.zeros(hkv, 0, dim, dtype=torch.float64, device=DEVICE)
    ids = state["table"][b, : -(-length // page)].long()
    got = state[side + "_pages"][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :length]
    if fmt == "none":
        return got.double()
    if FORMATS[fmt][1] + FORMATS[fmt][2] == 3:
        got = torch.stack([got.to(torch.int64) % 16, got.to(torch.int64) // 16], -1).flatten(-2)
    s = state[side + "_scales"][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :length].to(torch.int64) - 127
    return _value_of(got, fmt) * torch.ldexp(torch.ones_like(s, dtype=torch.float64), s).repeat_interleave(32, -1)


def _exact_quantized(x, fmt):
    """What rows x[..., dim] become in the cache, float64, from the definition of the format: nearest multiple of the
    step of the element's binade, ties to even, with the format's own rules at both ends of the range."""
    kind, e, f = FORMATS[fmt]
    if kind == "none":
        return x.to(torch.bfloat16).double()
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    v = blocks.double()
    if kind == "mxint":
        top = blocks.abs().amax(-1, keepdim=True).clamp(min=torch.finfo(x.dtype).tiny)
        unit = torch.exp2(torch.log2(top).ceil().double() - (e - 1))
        return (torch.round(v / unit).clamp(-(2 ** (e - 1)), 2 ** (e - 1) - 1) * unit).reshape(x.shape)
    bias, last = 2 ** (e - 1) - 1, 2 ** e - 1
    v = torch.where(v.abs() < 2.0 ** -126, 0.0, v)
    top = v.abs().amax(-1, keepdim=True)
    binade = lambda t: torch.frexp(t)[1].double() - 1  # noqa: E731
    shared = torch.where(top > 0, (binade(top) - (last - bias)).clamp(-127, 128), -127.0)
    field = binade(v.abs()) - shared + bias  # the exponent field an element of this size has
    low = torch.exp2(binade(v.abs()))
    m = torch.floor(v.abs() / low * 2 ** 15) - 2 ** 15  # 15 bits of the fraction
    q = torch.round(m / 2 ** (15 - f))                  # 0 .. 2^f
    # a fraction that rounds up to 2^f is OR-ed onto the exponent field: the carry is lost when the field is odd
    odd = torch.remainder(field, 2) == 1
    carried = q == 2 ** f
    whole = torch.where(carried & ~odd, torch.exp2(field + 1 - bias),
                        torch.where(carried, torch.exp2(field - bias), torch.exp2(field - bias) * (1 + q / 2 ** f)))
    sub = torch.where(q > 0, torch.floor(torch.where(carried, q, q + 2 ** f) / 2), q)
    tiny = torch.where(sub >= 2 ** f, torch.full_like(sub, 2.0 ** (1 - bias)), sub * 2.0 ** (1 - bias - f))
    out = torch.where(field > 0, whole, torch.where(field == 0, tiny, 0.0))
    out = torch.where(field > last, (2 - 2.0 ** -f) * 2.0 ** (last - bias), out)
    out = torch.where(v == 0, 0.0, out) * torch.exp2(shared)
    return (torch.sign(v) * out).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    op, n, hkv = case["op"], case["batch"], case["kv_heads"]
    lens = _lengths(case)
    if op == "evict":
        return _exact_evict(state, lens)
    new = _counts(case) if op == "prompt" else [1] * n if op == "step" else [0] * n
    sides = {}
    for side in ("key", "value"):
        rows = []
        for b in range(n):
            r = _exact_rows(state, side, b, lens[b])
            if new[b]:
                r = torch.cat([r, _exact_quantized(state[side][b, :, : new[b]].contiguous(), case["fmt"])], 1)
            rows.append(r)
        sides[side] = rows
    if op == "prompt":
        most = state["most"]
        return [torch.stack([torch.nn.functional.pad(r, (0, 0, 0, most - r.shape[1])) for r in sides[s]])
                for s in ("key", "value")]
    g = case["heads"] // hkv
    out, weights = [], state["weights"].double() if op == "tracked" else None
    for b in range(n):
        k, v = sides["key"][b], sides["value"][b]
        q = state["query"][b].double().view(hkv, g, case["dim"])
        p = torch.softmax(q @ k.transpose(1, 2) * state["scaling"], -1)
        out.append((p @ v).reshape(case["heads"], 1, case["dim"]))
        if weights is not None:
            weights[b, :, : lens[b]] += p.sum(1)
    out = torch.stack(out)
    return out if weights is None else (out, weights)


def _exact_evict(state, lens):
    case = state["case"]
    keep, page = case["keep"], case["page"]
    w, pos = state["weights"].double().cpu(), state["positions"].cpu()
    out_w, out_p = torch.zeros_like(w), torch.full_like(pos, -1)
    pages = {s: state[s + "_pages"].double() for s in ("key", "value")}
    table = state["table"].cpu()
    for b, length in enumerate(lens):
        for h in range(case["kv_heads"]):
            m = min(length, keep)
            safe = pos[b, h, :length] >= length - case["recent"]
            rank = torch.where(safe, math.inf, w[b, h, :length])
            kept = torch.sort(rank, descending=True, stable=True).indices[:m].sort().values
            stay, move = kept[kept < m], kept[kept >= m]
            place = torch.arange(m)
            free = torch.ones(m, dtype=torch.bool)
            free[stay] = False
            free = free.nonzero().view(-1)
            source = place.clone()
            source[free] = move
            out_w[b, h, :m], out_p[b, h, :m] = w[b, h, source], pos[b, h, source]
            if len(free):
                ids = lambda at: (table[b, at // page].long().to(DEVICE), h, (at % page).to(DEVICE))  # noqa: E731
                for s in pages:
                    pages[s][ids(free)] = pages[s][ids(move)]
    return (torch.tensor([min(x, keep) for x in lens], dtype=torch.float64), out_w, out_p, pages["key"], pages["value"])
