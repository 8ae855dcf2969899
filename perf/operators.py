"""The operators of a quantised decode path, as cases that can be timed and checked.

Rows quantised to 8-bit integers and the product of such rows with 8-bit weights, a paged
cache of keys and values held in 4 bits (written and read back), and attention over it,
as a program calls them on device-resident operands.  Where ``own`` is true ``run`` calls
``oct_amd.prometheus.NativeRuntime``; where it is false it computes the same with
elementary torch operations in 32 bits, rounded once at the end.

``listed()`` names the fixed cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes what a program has in hand before the call, ``run`` is one call,
``work`` the bytes and operations it cannot do without, ``exact`` the same result in 64
bits from the operators' definitions.

Definitions.  A row x in 8 bits: s = max |x| / 127 and q = rint(x / s), each operation
rounded to 32 bits.  The product: c[i, j] = a_scale[i] w_scale[j] sum_k a[i, k] w[j, k].
A group of 64 channels x in 4 bits: s = max |x| / 6, rounded to 32 bits and then up to six
significant bits; a channel is held as the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their
negatives to x / s (rounded to 32 bits; halfway to the even code), and stands for s times
that, a number of eight significant bits at most.  Attention: the new rows of a sequence are
its last ones; row r of position p sees the keys at positions max(0, p - window + 1)..p
(0..p without a window).

The cache is a pool of pages of 64 tokens.  A page holds, head after head, the keys' codes
[64][D / 2], the values' codes [64][D / 2], the keys' parameters [D / 64][64] and the
values'.  A code is a sign (8) and the place 0..7 of the magnitude in the list above; a byte
holds two channels, the lower one in its low half.  A value row lies in channel order; in a
key row, in blocks of 128 channels (64 for D = 64), the 4-byte word of channels 32 s + 8 h ..
+ 7 lies at word S h + s, S = block / 32.  A parameter is the upper 16 bits of s as a 32-bit
float.
"""
from __future__ import annotations

import math

import torch

own = False

F32, BF16 = "fp32", "bf16"
TYPES = {F32: torch.float32, BF16: torch.bfloat16}
PAGE = 64
GROUP = 64


def listed() -> list:
    return [
        # One token's hidden state before a decoder layer's products: the smallest call.
        {"name": "rows_int8_token", "kind": "rows", "rows": 1, "width": 2048, "type": BF16},
        # The gated hidden rows of the largest image block before its down projection.
        {"name": "rows_int8_image", "kind": "rows", "rows": 4224, "width": 10240, "type": BF16},
        # One token through a decoder layer's gate and up weights: the weights are read once.
        {"name": "int8_token", "kind": "product", "m": 1, "n": 32768, "k": 2048, "type": F32},
        # A short prompt through the same layer's down projection: few columns, long sums.
        {"name": "int8_tokens15", "kind": "product", "m": 15, "n": 2048, "k": 16384, "type": F32},
        # No side a multiple of a tile, two of them odd: data as it comes.
        {"name": "int8_ragged", "kind": "product", "m": 4097, "n": 3001, "k": 513, "type": F32},
        # The gate and up projection of the largest image block.
        {"name": "int8_image", "kind": "product", "m": 4224, "n": 20480, "k": 3840, "type": BF16},
        # One new token of each of 64 conversations goes into the cache and is read back.
        {"name": "kv4_append", "kind": "cache", "sequences": 64, "longest": 4096, "new": 1, "heads": 8, "dim": 128,
         "type": BF16},
        # Prompts of uneven lengths fill an empty cache and are read back.
        {"name": "kv4_prompts", "kind": "cache", "sequences": 5, "longest": 8191, "new": 8191, "heads": 8, "dim": 128,
         "type": BF16},
        # One token of a short conversation on a decoder with a single key head.
        {"name": "attention_token", "kind": "attention", "sequences": 1, "longest": 777, "new": 1, "heads": 1,
         "group": 8, "dim": 256, "window": 0, "type": F32},
        # A step of 64 conversations of uneven lengths.
        {"name": "attention_batch", "kind": "attention", "sequences": 64, "longest": 8192, "new": 1, "heads": 8,
         "group": 4, "dim": 128, "window": 0, "type": BF16},
        # One token at the end of a very long document.
        {"name": "attention_long", "kind": "attention", "sequences": 1, "longest": 131072, "new": 1, "heads": 8,
         "group": 4, "dim": 128, "window": 0, "type": BF16},
        # Pieces of prompts over what their conversations hold already.
        {"name": "attention_prompts", "kind": "attention", "sequences": 4, "longest": 8000, "new": 1024, "heads": 8,
         "group": 4, "dim": 128, "window": 0, "type": BF16},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("rows", "product", "product", "cache", "attention", "attention", "attention"))
    dtype = rng.choice((F32, BF16))
    if kind == "rows":
        rows = _log_int(rng, 1, 8192)
        width = _log_int(rng, 64, min(16384, (1 << 25) // rows))
        return {"kind": kind, "rows": rows, "width": width // 128 * 128 if rng.random() < 0.5 and width > 128 else width,
                "type": dtype}
    if kind == "product":
        m, n = _log_int(rng, 1, 4224), _log_int(rng, 256, 20480)
        k = _log_int(rng, 128, min(16384, 300_000_000_000 // (m * n)))
        if rng.random() < 0.6:  # most models' widths are multiples of 128
            n, k = n // 128 * 128, k // 128 * 128
        return {"kind": kind, "m": m, "n": n, "k": k, "type": dtype}
    dim = rng.choice((64, 128, 256))
    heads = rng.choice((1, 2, 5, 8))
    if kind == "cache":
        new = rng.choice((1, _log_int(rng, 2, 8192)))
        sequences = min(_log_int(rng, 1, 128), max(1, 20000 // new))
        return {"kind": kind, "sequences": sequences, "longest": new + _log_int(rng, 1, 4096), "new": new,
                "heads": heads, "dim": dim, "type": dtype}
    group = rng.choice((1, 3, 4, 8, 16))
    if rng.random() < 0.6:
        new, sequences = 1, _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, 60_000_000 // (sequences * heads * dim))
    else:
        new, sequences = _log_int(rng, 2, 1024), _log_int(rng, 1, 4)
        longest = new + _log_int(rng, 1, 8192)
        group = min(group, 4)
    return {"kind": kind, "sequences": sequences, "longest": min(longest, 131072), "new": new, "heads": heads,
            "group": group, "dim": dim, "window": rng.choice((0, 0, _log_int(rng, 16, 4096))), "type": dtype}


# ------------------------------------------------------------------ lengths
def _spread(count: int, lo: int, hi: int) -> list:
    """`count` uneven numbers of lo..hi, the first of them hi."""
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(count)]


def _new_rows(case) -> list:
    return _spread(case["sequences"], min(case["new"], 1 + case["new"] // 8), case["new"])


def _lengths(case) -> list:
    """Tokens of each sequence after the call, its new rows among them."""
    new = _new_rows(case)
    old = max(0, case["longest"] - case["new"])
    return [n + o for n, o in zip(new, _spread(case["sequences"], old // 8, old))]


# ------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(std) if std != 1.0 else t


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _key_rows(g, shape):
    """Keys as projections give them: a few channels of each head are several times larger."""
    x = _normal(g, shape)
    x[..., ::37] *= 4.0
    return x


def _product_inputs(case, g) -> dict:
    m, n, k = case["m"], case["n"], case["k"]
    whole = lambda *shape: torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    scale = lambda count, top: torch.rand(count, generator=g, device="cuda").mul_(top).add_(0.1 * top)  # noqa: E731
    return {"a": whole(m, k), "w": whole(n, k), "a_scale": scale(m, 0.03), "w_scale": scale(n, 0.0005)}


def _cache_inputs(case, g) -> dict:
    """New rows, and for attention the rows that the cache holds, in the order of sequences and positions."""
    heads, dim, dtype = case["heads"], case["dim"], TYPES[case["type"]]
    rows = sum(_new_rows(case))
    held = rows if case["kind"] == "cache" else sum(_lengths(case))
    x = {"k": _key_rows(g, (held, heads, dim)).to(dtype), "v": _normal(g, (held, heads, dim)).to(dtype)}
    if case["kind"] == "attention":
        x["q"] = _normal(g, (rows, heads * case["group"], dim)).to(dtype)
    return x


def _inputs(case, seed) -> dict:
    g = _generator(seed)
    if case["kind"] == "rows":
        return {"x": _normal(g, (case["rows"], case["width"])).to(TYPES[case["type"]])}
    return _product_inputs(case, g) if case["kind"] == "product" else _cache_inputs(case, g)


def _places(lengths: torch.Tensor, counts: torch.Tensor, rows: int):
    """Sequence and position of each of `rows` packed rows, the last counts[i] of sequence i."""
    counts = counts.long()
    sequence = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=rows)
    first = torch.cumsum(counts, 0) - counts
    row = torch.arange(rows, device="cuda")
    return sequence, row - first[sequence] + (lengths.long() - counts)[sequence]


def prepare(case, seed) -> dict:
    s = dict(_inputs(case, seed), case=case)
    if case["kind"] == "rows":
        s["q"] = torch.empty((case["rows"], case["width"]), dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
    elif case["kind"] == "product":
        s["c"] = torch.empty((case["m"], case["n"]), dtype=TYPES[case["type"]], device="cuda")
    else:
        lengths, new = _lengths(case), _new_rows(case)
        counts = [-(-n // PAGE) for n in lengths]
        s["pages"], s["table_stride"], s["rows"] = sum(counts) + 3, max(counts), sum(new)
        # Pages are handed out in no order; the rest of a sequence's table is not used.
        order = torch.randperm(s["pages"], generator=_generator(seed + 1), device="cuda")
        used = torch.arange(max(counts), device="cuda") < _ints(counts)[:, None]
        table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
        table[used] = order[:sum(counts)].int()
        s["table"], s["lengths"], s["new"] = table, _ints(lengths), _ints(new)
        s["row_starts"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["pool"] = torch.zeros((s["pages"], case["heads"], _block_bytes(case["dim"])), dtype=torch.uint8, device="cuda")
        if case["kind"] == "cache":
            s["k_read"], s["v_read"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        else:
            sequence, position = _places(s["lengths"], s["lengths"], sum(lengths))
            _store(s, s.pop("k"), s.pop("v"), sequence, position)
            s["out"] = torch.empty_like(s["q"])
    # The reactor works on its own stream: what torch still has queued comes first.
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_rows(s):
    x = s["x"].float()
    scale = x.abs().amax(-1) / torch.full_like(x[:, 0], 127.0)
    q = torch.round(x / scale[:, None]).nan_to_num_(0.0)
    return {"q": q.to(torch.int8), "scale": scale}


def _plain_product(s):
    c = s["a"].float() @ s["w"].float().t().contiguous()
    return (c * s["a_scale"][:, None] * s["w_scale"]).to(s["c"].dtype)


def _block_bytes(dim: int) -> int:
    return PAGE * dim + 4 * PAGE * (dim // GROUP)


def _regions(s):
    """The pool's key codes, value codes [page, head, token, D / 2] and parameters [page, head, D / 64, token]."""
    pool, dim, heads = s["pool"], s["case"]["dim"], s["case"]["heads"]
    half, codes = PAGE * dim // 2, (s["pages"], heads, PAGE, dim // 2)
    groups = (s["pages"], heads, dim // GROUP, PAGE)
    span = 2 * PAGE * (dim // GROUP)
    params = pool[..., 2 * half:].view(torch.int16)
    return (pool[..., :half].view(codes), pool[..., half:2 * half].view(codes),
            params[..., :span // 2].view(groups), params[..., span // 2:].view(groups))


def _quantise(x):
    """Codes [rows, heads, D] and parameters [rows, heads, D / 64] of the groups of x."""
    g = x.float().unflatten(-1, (-1, GROUP))
    step = g.abs().amax(-1)
    step = step / torch.full_like(step, 6.0)
    step = ((step.view(torch.int32) + 0x3FFFF) & -0x40000).view(torch.float32)
    y = (g / step[..., None]).nan_to_num_(0.0)
    # The borders between the magnitudes; a border itself goes to the even one of its neighbours.
    up = torch.tensor([0.75, 1.75, 3.5], device="cuda")
    down = torch.tensor([0.25, 1.25, 2.5, 5.0], device="cuda")
    a = y.abs()
    code = torch.bucketize(a, up, right=True).add_(torch.bucketize(a, down))
    code = torch.where(y < 0.0, code + 8, code)
    return code.to(torch.uint8).flatten(-2), (step.view(torch.int32) >> 16).to(torch.int16)


def _key_order(n, dim: int, back: bool):
    block = min(dim, 128)
    shape = (dim // block, 4, block // 32, 8) if back else (dim // block, block // 32, 4, 8)
    return n.unflatten(-1, shape).transpose(-3, -2).flatten(-4)


def _store(s, k, v, sequence, position):
    dim = s["case"]["dim"]
    page, slot = s["table"][sequence, position // PAGE].long(), position % PAGE
    keys, values, key_params, value_params = _regions(s)
    kn, kp = _quantise(k)
    vn, vp = _quantise(v)
    kn = _key_order(kn, dim, False)
    keys[page, :, slot] = kn[..., 0::2] | (kn[..., 1::2] << 4)
    values[page, :, slot] = vn[..., 0::2] | (vn[..., 1::2] << 4)
    key_params[page, :, :, slot] = kp
    value_params[page, :, :, slot] = vp


def _values(codes):
    """The numbers that codes [..., D / 2] name, in stored order."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    names = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    return torch.cat((names, -names))[n]


def _load(s, page, slot):
    """Keys and values [..., heads, D] in 32 bits of the tokens at `slot` of `page` (indices of one shape)."""
    dim = s["case"]["dim"]
    keys, values, key_params, value_params = _regions(s)
    step = lambda params: (params[page, :, :, slot].int() << 16).view(torch.float32)[..., None]  # noqa: E731
    k = _key_order(_values(keys[page, :, slot]), dim, True).unflatten(-1, (-1, GROUP)) * step(key_params)
    v = _values(values[page, :, slot]).unflatten(-1, (-1, GROUP)) * step(value_params)
    return k.flatten(-2), v.flatten(-2)


def _plain_cache(s):
    sequence, position = _places(s["lengths"], s["new"], s["rows"])
    _store(s, s["k"], s["v"], sequence, position)
    k, v = _load(s, s["table"][sequence, position // PAGE].long(), position % PAGE)
    return {"k": k.to(s["k"].dtype), "v": v.to(s["v"].dtype)}


def _plain_attention(s):
    case = s["case"]
    heads, group, dim, sequences = case["heads"], case["group"], case["dim"], case["sequences"]
    lengths, new = s["lengths"].long(), s["new"].long()
    # Every sequence's keys and values, padded to the longest: [sequences, heads, longest, D].
    key = torch.arange(s["table_stride"] * PAGE, device="cuda")
    page = s["table"].long().clamp(min=0)[:, key // PAGE]
    k, v = _load(s, page, (key % PAGE).expand_as(page))
    held = (key < lengths[:, None])[:, :, None, None]
    k, v = (torch.where(held, t, 0.0).transpose(1, 2).contiguous() for t in (k, v))
    # Its rows, padded to the most: [sequences, heads, rows * group, D].
    row = torch.arange(case["new"], device="cuda")
    live = row < new[:, None]
    at = (s["row_starts"].long()[:-1, None] + row).clamp(max=s["rows"] - 1)
    q = s["q"].float()[at].view(sequences, case["new"], heads, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(sequences, heads, -1, dim)
    position = (lengths - new)[:, None] + row
    seen = key <= position[..., None]
    if case["window"]:
        seen &= key > position[..., None] - case["window"]
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = (q @ k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(dim)).masked_fill_(~seen, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    out = (p @ v) / p.sum(-1, keepdim=True)
    out = out.view(sequences, heads, case["new"], group, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(sequences, case["new"], heads * group, dim)[live].to(s["q"].dtype)


# ------------------------------------------------------------------ the framework's operators
_runtime = None


def _reactor():
    """The module and the one runtime handle a program opens and keeps."""
    global _runtime
    from oct_amd import prometheus as p

    if _runtime is None:
        _runtime = p.NativeRuntime()
        _runtime.require_hardware_gpu()
    return p, _runtime


def _own(s):
    p, rt = _reactor()
    case = s["case"]
    dtype = p.DTYPE_BF16 if case["type"] == BF16 else p.DTYPE_F32
    if case["kind"] == "rows":
        rt.quantize_rows_int8_device(s["x"].data_ptr(), s["q"].data_ptr(), s["scale"].data_ptr(), case["rows"],
                                     case["width"], case["width"], dtype)
        return {"q": s["q"], "scale": s["scale"]}
    if case["kind"] == "product":
        rt.gemm_int8_device(s["a"].data_ptr(), s["w"].data_ptr(), s["a_scale"].data_ptr(), s["w_scale"].data_ptr(),
                            s["c"].data_ptr(), case["m"], case["n"], case["k"], dtype)
        return s["c"]
    cache = p.kv4_cache(s["pool"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(), case["dim"],
                        case["heads"], s["pages"], case["sequences"], s["table_stride"])
    if case["kind"] == "cache":
        stride = case["heads"] * case["dim"]
        rt.kv4_write_device(cache, s["k"].data_ptr(), s["v"].data_ptr(), s["row_starts"].data_ptr(), s["rows"], stride,
                            dtype)
        rt.kv4_read_device(cache, s["k_read"].data_ptr(), s["v_read"].data_ptr(), s["row_starts"].data_ptr(),
                           s["rows"], stride, dtype)
        return {"k": s["k_read"], "v": s["v_read"]}
    q_heads = case["heads"] * case["group"]
    rt.attention_kv4_device(cache, s["q"].data_ptr(), s["out"].data_ptr(), s["row_starts"].data_ptr(), s["rows"],
                            q_heads, q_heads * case["dim"], q_heads * case["dim"], case["new"], case["longest"],
                            case["window"], 1.0 / math.sqrt(case["dim"]), dtype)
    return s["out"]


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "rows":
        return _plain_rows(s)
    if kind == "product":
        return _plain_product(s)
    return _plain_cache(s) if kind == "cache" else _plain_attention(s)


def work(case) -> dict:
    size = 4 if case["type"] == F32 else 2
    if case["kind"] == "rows":
        rows, width = case["rows"], case["width"]
        return {"bytes": rows * width * (size + 1) + 4 * rows, "flops": 3 * rows * width}
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + size * m * n, "flops": 2 * m * n * k}
    heads, dim = case["heads"], case["dim"]
    token = heads * (dim + 4 * (dim // GROUP))  # one token's keys and values in the cache
    new = _new_rows(case)
    if case["kind"] == "cache":
        # rows in, into the cache, out of it, and out
        return {"bytes": sum(new) * (4 * heads * dim * size + 2 * token), "flops": 16 * sum(new) * heads * dim}
    window = case["window"] or 1 << 40
    held = seen = 0
    for n, length in zip(new, _lengths(case)):
        held += min(length, window + n - 1)
        seen += sum(min(p + 1, window) for p in range(length - n, length))
    q_heads = heads * case["group"]
    return {"bytes": held * token + 2 * sum(new) * q_heads * dim * size, "flops": 4 * seen * q_heads * dim}


# ------------------------------------------------------- the same in 64 bits
def _to32(x):
    """One rounding to 32 bits, as the definitions ask of a quotient."""
    return x.to(torch.float32).to(torch.float64)


def _exact_values(x):
    """What the groups of x are held as, value by value from the definition."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    # mantissa in [1/2, 1): six significant bits are 64ths of the power of two above
    mantissa, exponent = torch.frexp(_to32(g.abs().max(-1)[0] / 6.0))
    step = torch.ldexp(torch.ceil(mantissa * 64.0) / 64.0, exponent)[..., None]
    y = torch.where(step > 0.0, _to32(g / step), 0.0)
    # The distance between neighbours doubles at 2 and at 4, and an even multiple of it is an even code.
    unit = torch.where(y.abs() < 2.0, 0.5, torch.where(y.abs() < 4.0, 1.0, 2.0))
    return (step * (torch.round(y / unit) * unit)).reshape(x.shape)


def _exact_attention(case, x):
    heads, group, dim = case["heads"], case["group"], case["dim"]
    lengths, new = _lengths(case), _new_rows(case)
    k, v = _exact_values(x["k"]), _exact_values(x["v"])
    out = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    first_key = first_row = 0
    for length, rows in zip(lengths, new):
        position = torch.arange(length - rows, length, device="cuda")
        key = torch.arange(length, device="cuda")
        hidden = key[None, :] > position[:, None]
        if case["window"]:
            hidden |= key[None, :] <= position[:, None] - case["window"]
        for h in range(heads):
            kh, vh = (t[first_key:first_key + length, h].contiguous() for t in (k, v))
            for j in range(h * group, (h + 1) * group):
                q = x["q"][first_row:first_row + rows, j].double()
                scores = (q @ kh.t().contiguous() / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                out[first_row:first_row + rows, j] = torch.softmax(scores, -1) @ vh
        first_key += length
        first_row += rows
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "rows":
        rows = x["x"].double()
        scale = _to32(rows.abs().max(-1)[0] / 127.0)
        return {"q": torch.round(_to32(rows / scale[:, None])).to(torch.int8), "scale": scale}
    if case["kind"] == "product":
        c = x["a"].double() @ x["w"].double().t().contiguous()
        return c * (x["a_scale"].double()[:, None] * x["w_scale"].double()[None, :])
    if case["kind"] == "cache":
        return {"k": _exact_values(x["k"]), "v": _exact_values(x["v"])}
    return _exact_attention(case, x)
