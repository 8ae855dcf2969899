"""The rest of a decoder's step beside its quantised path, as cases that can be timed and checked.

Weights held in 4 bits with a step for each group (packed and unpacked), products of rows
with such weights, a whole mixture-of-experts layer on them, rotary positions, and the
residual sum between two blocks with the norms before and after it.  Where ``own`` is true
``run`` calls ``oct_amd.prometheus.NativeRuntime``; where it is false it computes the same
with elementary torch operations in 32 bits, rounded once at the end.

``listed()`` names the fixed cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes what a program has in hand before the call, ``run`` is one call,
``work`` the bytes and operations it cannot do without, ``exact`` the same result in 64
bits from the operators' definitions.

Definitions.  A weight matrix w [n, k] in 4 bits: a group is `group` neighbouring weights of
a row (fewer at its end); s = max |w| / 6, rounded to 32 bits and then up to six significant
bits; a weight is held as the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives to
w / s (rounded to 32 bits; halfway to the even code), and stands for s times that, a number of
eight significant bits at most.  The product: c[i, j] = sum_k x[i, k] w[j, k].

A mixture: l = x router^T in 64 bits; a token's experts are the top_k of the largest l, in that
order (ties to the lower expert); p = softmax(l) over all experts, divided by the sum over the
chosen ones where `renormalise` is set; out = sum over the chosen e of p_e
(act(x gate_e^T) * (x up_e^T)) down_e^T with act SiLU or the tanh form of GELU.

Rotary positions: the first `rotary` channels of each head, in pairs (i, i + rotary / 2)
("half") or (2 i, 2 i + 1) ("pairs"), are turned by position * frequency_i and scaled by a
magnitude; the other channels stay.  frequency_i = base^(-2 i / rotary), scaled for longer
contexts: "linear" divides all by `factor`; "base" takes base * factor^(rotary / (rotary - 2));
"parts" divides those that turn less than once within `context` tokens, keeps those that turn
32 times or more, goes linearly over i between, and has magnitude 1 + ln(factor) / 10.

A residual sum with norms: h' = h + residual_scale * gate * norm(y; post), out = norm(h'; pre)
* (1 + scale) + shift; norm(x; w) = x / sqrt(mean(x^2) + eps) * w; gate (its tanh), scale and
shift are rows that `per` neighbouring rows share.

The packed matrix: tiles of 16 rows by 128 columns, in each row of tiles those of rising
columns.  A tile's codes are 64 times 16 bytes: the 16 bytes of lane l are four words, word s
the codes of row l % 16, columns 32 s + 8 (l / 16) .. + 7, the lower column in the lower half of
a byte; a code is a sign (8) and the place 0..7 of the magnitude in the list above.  Behind all
codes lie the steps, tile by tile, [16][128 / group], each the upper 16 bits of a 32-bit float.
Rows and columns behind the last are zeros.
"""
from __future__ import annotations

import math

import torch

own = False

F32, BF16 = "fp32", "bf16"
TYPES = {F32: torch.float32, BF16: torch.bfloat16}
TILE_N, TILE_K = 16, 128
SILU, GELU = "silu", "gelu"
EPS = 1e-6


def listed() -> list:
    return [
        # A weight matrix of sides that are not whole tiles, laid out when a model is loaded.
        {"name": "w4_pack_ragged", "kind": "pack", "n": 1001, "k": 651, "group": 32, "type": F32},
        # A decoder layer's gate weights at load time.
        {"name": "w4_pack_gate", "kind": "pack", "n": 16384, "k": 2048, "group": 128, "type": BF16},
        # One token through a decoder layer's gate and up weights: the weights are read once.
        {"name": "w4_token", "kind": "product", "m": 1, "n": 32768, "k": 2048, "group": 128, "type": BF16},
        # A short prompt through the down projection in fp32: few columns, long sums.
        {"name": "w4_tokens15", "kind": "product", "m": 15, "n": 2048, "k": 16384, "group": 32, "type": F32},
        # A batch of conversations on sides that are not whole tiles.
        {"name": "w4_ragged", "kind": "product", "m": 33, "n": 3001, "k": 1999, "group": 64, "type": BF16},
        # A prompt through the gate and up projection of the image model's width.
        {"name": "w4_prompt", "kind": "product", "m": 512, "n": 20480, "k": 3840, "group": 64, "type": BF16},
        # One token through a mixture: eight experts' weights are read.
        {"name": "moe_token", "kind": "mixture", "tokens": 1, "hidden": 2048, "inner": 1024, "experts": 64, "top_k": 8,
         "group": 32, "act": SILU, "renormalise": True, "type": BF16},
        # A step of 64 conversations: nearly every expert has some tokens.
        {"name": "moe_batch", "kind": "mixture", "tokens": 64, "hidden": 2048, "inner": 1024, "experts": 64, "top_k": 8,
         "group": 64, "act": GELU, "renormalise": False, "type": BF16},
        # One token's queries and its single key head, far into a document.
        {"name": "rope_token", "kind": "rope", "rows": 1, "q_heads": 8, "k_heads": 1, "dim": 256, "rotary": 256,
         "layout": "half", "scaling": "none", "factor": 1.0, "context": 8192, "first": 100000, "type": F32},
        # A whole prompt, half of each head, in a context eight times the trained one.
        {"name": "rope_prompt", "kind": "rope", "rows": 8191, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 64,
         "layout": "pairs", "scaling": "parts", "factor": 8.0, "context": 4096, "first": 0, "type": BF16},
        # One token between a decoder's attention and its feed-forward.
        {"name": "norm_token", "kind": "norm", "rows": 1, "width": 2048, "post": True, "gate": False, "modulate": False,
         "per": 1, "residual_scale": 1.0, "type": F32},
        # An image block's gated residual with its modulated norm.
        {"name": "norm_image", "kind": "norm", "rows": 4224, "width": 3840, "post": True, "gate": True,
         "modulate": True, "per": 4224, "residual_scale": 1.0, "type": BF16},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("pack", "product", "product", "product", "mixture", "mixture", "mixture", "rope", "norm"))
    dtype = rng.choice((F32, BF16))
    group = rng.choice((32, 64, 128))
    if kind == "pack":
        n = _log_int(rng, 16, 16384)
        return {"kind": kind, "n": n, "k": _log_int(rng, 64, min(16384, 33_000_000 // n)), "group": group, "type": dtype}
    if kind == "product":
        m = _log_int(rng, 65, 512) if rng.random() < 0.2 else _log_int(rng, 1, 64)
        n = _log_int(rng, 256, 32768)
        k = _log_int(rng, 128, min(16384, 67_000_000 // n, 40_000_000_000 // (m * n)))
        if rng.random() < 0.6:  # most models' widths are multiples of 128
            n, k = n // 128 * 128, k // 128 * 128
        return {"kind": kind, "m": m, "n": n, "k": k, "group": group, "type": dtype}
    if kind == "mixture":
        hidden, inner = _log_int(rng, 256, 4096), _log_int(rng, 64, 2048)
        experts = _log_int(rng, 2, min(128, 400_000_000 // (3 * hidden * inner)))
        if rng.random() < 0.6:
            hidden, inner = hidden // 128 * 128, max(64, inner // 64 * 64)
        return {"kind": kind, "tokens": rng.choice((1, _log_int(rng, 2, 64))), "hidden": hidden, "inner": inner,
                "experts": experts, "top_k": rng.randint(1, min(8, experts)), "group": group,
                "act": rng.choice((SILU, GELU)), "renormalise": rng.random() < 0.5, "type": dtype}
    if kind == "rope":
        dim = rng.choice((64, 80, 128, 256))
        k_heads = rng.choice((1, 2, 5, 8))
        q_heads = k_heads * rng.choice((1, 3, 4, 8))
        rows = _log_int(rng, 1, min(8192, 42_000_000 // ((q_heads + k_heads) * dim)))
        return {"kind": kind, "rows": rows, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
                "rotary": rng.choice((dim, dim // 2, dim // 4 + dim // 4 % 2)), "layout": rng.choice(("half", "pairs")),
                "scaling": rng.choice(("none", "linear", "base", "parts")), "factor": rng.choice((2.0, 8.0, 32.0)),
                "context": rng.choice((2048, 4096, 8192)), "first": rng.choice((0, _log_int(rng, 1, 1_000_000))),
                "type": dtype}
    width = _log_int(rng, 64, 16384)
    rows = _log_int(rng, 1, min(8192, 16_000_000 // width))
    return {"kind": "norm", "rows": rows, "width": width // 128 * 128 if rng.random() < 0.5 and width > 128 else width,
            "post": rng.random() < 0.6, "gate": rng.random() < 0.5, "modulate": rng.random() < 0.5,
            "per": rng.choice((1, _log_int(rng, 1, rows))), "residual_scale": rng.choice((1.0, 0.22)), "type": dtype}


# ------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(std) if std != 1.0 else t


def _weights(g, n, k):
    """A projection's weights: rows that keep the size of what they multiply, a few channels larger."""
    w = _normal(g, (n, k), 1.0 / math.sqrt(k))
    w[:, ::53] *= 3.0
    return w


def _expert_shapes(case):
    hidden, inner = case["hidden"], case["inner"]
    return {"gate": (inner, hidden), "up": (inner, hidden), "down": (hidden, inner)}


def _experts(case, seed):
    """One expert's three weight matrices after the other."""
    g = _generator(seed + 1)
    for _ in range(case["experts"]):
        yield {name: _weights(g, *shape) for name, shape in _expert_shapes(case).items()}


def _inputs(case, seed) -> dict:
    g = _generator(seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    if kind == "pack":
        return {"w": _weights(g, case["n"], case["k"]).to(dtype)}
    if kind == "product":
        return {"x": _normal(g, (case["m"], case["k"])).to(dtype), "w": _weights(g, case["n"], case["k"])}
    if kind == "mixture":
        return {"x": _normal(g, (case["tokens"], case["hidden"])).to(dtype),
                "router": _normal(g, (case["experts"], case["hidden"]), 1.5 / math.sqrt(case["hidden"]))}
    if kind == "rope":
        rows, dim = case["rows"], case["dim"]
        jump = torch.randint(0, 97, (1,), generator=g, device="cuda", dtype=torch.int32)
        return {"q": _normal(g, (rows, case["q_heads"], dim)).to(dtype),
                "k": _normal(g, (rows, case["k_heads"], dim)).to(dtype),
                "positions": torch.arange(rows, dtype=torch.int32, device="cuda") + case["first"] + jump}
    rows, width, shared = case["rows"], case["width"], -(-case["rows"] // case["per"])
    x = {"h": _normal(g, (rows, width), 3.0).to(dtype), "y": _normal(g, (rows, width), 0.7).to(dtype),
         "pre": _normal(g, (width,), 0.1).add_(1.0)}
    if case["post"]:
        x["post"] = _normal(g, (width,), 0.1).add_(1.0)
    if case["gate"]:
        x["gate"] = _normal(g, (shared, width)).to(dtype)
    if case["modulate"]:
        x["scale"], x["shift"] = (_normal(g, (shared, width), 0.3).to(dtype) for _ in range(2))
    return x


def _frequencies(case):
    """Frequencies in radians a token (64 bits) and the magnitude."""
    rotary, factor, base, kind = case["rotary"], case["factor"], 10000.0, case["scaling"]
    if kind == "base":
        base *= factor ** (rotary / max(1, rotary - 2))
    i = torch.arange(rotary // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rotary)
    if kind == "linear":
        return f / factor, 1.0
    if kind != "parts":
        return f, 1.0
    # The pair that turns `turns` times within the trained context: base^(2 i / rotary) = context / (2 pi turns).
    at = lambda turns: rotary * math.log(case["context"] / (2.0 * math.pi * turns)) / (2.0 * math.log(base))  # noqa: E731
    low, high = max(0.0, math.floor(at(32.0))), min(rotary - 1.0, math.ceil(at(1.0)))
    slow = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    return f * (1.0 - slow) + f / factor * slow, 1.0 + 0.1 * math.log(factor)


def _matrix_bytes(n: int, k: int, group: int) -> int:
    return -(-n // TILE_N) * -(-k // TILE_K) * (TILE_N * TILE_K // 2 + 2 * TILE_N * (TILE_K // group))


def prepare(case, seed) -> dict:
    x = _inputs(case, seed)
    s = dict(x, case=case)
    kind, dtype, group = case["kind"], TYPES[case["type"]], case.get("group")
    empty = lambda *shape, dtype=dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if kind == "pack":
        s["packed"] = empty(_matrix_bytes(case["n"], case["k"], group), dtype=torch.uint8)
        s["out"] = torch.empty_like(s["w"])
    elif kind == "product":
        s["packed"] = _pack(s.pop("w"), group)
        s["out"] = empty(case["m"], case["n"])
    elif kind == "mixture":
        for name, (n, k) in _expert_shapes(case).items():
            s[name] = empty(case["experts"], _matrix_bytes(n, k, group), dtype=torch.uint8)
        for e, w in enumerate(_experts(case, seed)):
            for name in w:
                s[name][e] = _pack(w[name], group)
        s["out"] = torch.empty_like(s["x"])
        s["chosen"] = empty(case["tokens"], case["top_k"], dtype=torch.int32)
        s["weights"] = empty(case["tokens"], case["top_k"], dtype=torch.float32)
    elif kind == "rope":
        frequencies, s["magnitude"] = _frequencies(case)
        s["turns"] = (frequencies / (2.0 * math.pi)).to("cuda")  # revolutions a token
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    else:
        s["h_out"], s["out"] = torch.empty_like(s["h"]), torch.empty_like(s["h"])
    # The reactor works on its own stream: what torch still has queued comes first.
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the plain forms
def _quantise(w, group):
    """Codes [n, K] and steps [n, K / group] of rows padded to whole tiles."""
    w = w.float()
    padded = torch.zeros((-(-w.shape[0] // TILE_N) * TILE_N, -(-w.shape[1] // TILE_K) * TILE_K), device="cuda")
    padded[:w.shape[0], :w.shape[1]] = w
    g = padded.unflatten(-1, (-1, group))
    step = g.abs().amax(-1)
    step = step / torch.full_like(step, 6.0)
    step = ((step.view(torch.int32) + 0x3FFFF) & -0x40000).view(torch.float32)
    y = (g / step[..., None]).nan_to_num_(0.0)
    # The borders between the magnitudes; a border itself goes to the even one of its neighbours.
    up = torch.tensor([0.75, 1.75, 3.5], device="cuda")
    down = torch.tensor([0.25, 1.25, 2.5, 5.0], device="cuda")
    a = y.abs()
    code = torch.bucketize(a, up, right=True, out_int32=True).add_(torch.bucketize(a, down, out_int32=True))
    code = torch.where(y < 0.0, code + 8, code)
    return code.to(torch.uint8).flatten(-2), (step.view(torch.int32) >> 16).to(torch.int16)


def _pack(w, group):
    codes, steps = _quantise(w, group)
    tiles = codes.view(codes.shape[0] // TILE_N, TILE_N, codes.shape[1] // TILE_K, 4, 4, 8)
    tiles = tiles[..., 0::2] | (tiles[..., 1::2] << 4)
    tiles = tiles.permute(0, 2, 4, 1, 3, 5).reshape(-1)  # row tile, column tile, eighth of 32, row, 32, byte
    steps = steps.view(-1, TILE_N, codes.shape[1] // TILE_K, TILE_K // group).transpose(1, 2).reshape(-1)
    return torch.cat((tiles, steps.view(torch.uint8)))


def _unpack(packed, n, k, group):
    """The numbers [n, k] in 32 bits that a packed matrix stands for."""
    rows, cols = -(-n // TILE_N), -(-k // TILE_K)
    codes, steps = packed.split((rows * cols * TILE_N * TILE_K // 2, rows * cols * 2 * TILE_N * (TILE_K // group)))
    codes = codes.view(rows, cols, 4, TILE_N, 4, 4)
    names = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    v = torch.cat((names, -names))[torch.stack((codes & 15, codes >> 4), -1).int()]  # ..., word, byte, half
    v = v.flatten(-2).permute(0, 3, 1, 4, 2, 5).reshape(rows * TILE_N, cols * TILE_K // group, group)
    steps = (steps.view(torch.int16).int() << 16).view(torch.float32)
    steps = steps.view(rows, cols, TILE_N, TILE_K // group).transpose(1, 2).reshape(rows * TILE_N, -1)
    return (v * steps[..., None]).flatten(-2)[:n, :k]


def _times(x, w):
    """x w^T in 32 bits."""
    return x @ w.t().contiguous()


def _plain_pack(s):
    case = s["case"]
    s["packed"].copy_(_pack(s["w"], case["group"]))
    return _unpack(s["packed"], case["n"], case["k"], case["group"]).to(s["w"].dtype)


def _plain_product(s):
    case = s["case"]
    return _times(s["x"].float(), _unpack(s["packed"], case["n"], case["k"], case["group"])).to(s["out"].dtype)


def _activation(act, g):
    if act == SILU:
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_mixture(s):
    case = s["case"]
    x, experts, top_k = s["x"].float(), case["experts"], case["top_k"]
    # In 64 bits: two experts' logits may be close.
    logits = s["x"].double() @ s["router"].double().t().contiguous()
    order = torch.sort(logits, dim=-1, descending=True, stable=True)[1]
    chosen = order[:, :top_k]
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    picked = p.gather(1, chosen)
    weights = (picked / (picked if case["renormalise"] else p).sum(-1, keepdim=True)).float()
    dense = torch.zeros(x.shape[0], experts, device="cuda").scatter_(1, chosen, weights)
    out = torch.zeros_like(x)
    for e in range(experts):
        w = {name: _unpack(s[name][e], n, k, case["group"]) for name, (n, k) in _expert_shapes(case).items()}
        hidden = _activation(case["act"], _times(x, w["gate"])) * _times(x, w["up"])
        out += dense[:, e:e + 1] * _times(hidden, w["down"])
    return {"out": out.to(s["out"].dtype), "chosen": chosen.int(), "weights": weights}


def _plain_rope(s):
    case = s["case"]
    rotary, half = case["rotary"], case["rotary"] // 2
    # In 64 bits: a far position is many turns.
    turn = s["positions"].double()[:, None] * s["turns"]
    angle = (turn - torch.round(turn)) * (2.0 * math.pi)
    cos = (torch.cos(angle) * s["magnitude"]).float()[:, None]
    sin = (torch.sin(angle) * s["magnitude"]).float()[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        y = x.clone()
        if case["layout"] == "half":
            a, b = x[..., :half], x[..., half:rotary]
            y[..., :half], y[..., half:rotary] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
            y[..., 0:rotary:2], y[..., 1:rotary:2] = a * cos - b * sin, b * cos + a * sin
        out[name] = y.to(s[name].dtype)
    return out


def _plain_norm(s):
    case = s["case"]
    h, y = s["h"].float(), s["y"].float()
    norm = lambda x, w: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    rows = torch.arange(case["rows"], device="cuda") // case["per"]
    if case["post"]:
        y = norm(y, s["post"])
    if case["gate"]:
        y = y * torch.tanh(s["gate"].float())[rows]
    h = h + case["residual_scale"] * y
    out = norm(h, s["pre"])
    if case["modulate"]:
        out = out * (1.0 + s["scale"].float())[rows] + s["shift"].float()[rows]
    return {"h": h.to(s["h"].dtype), "out": out.to(s["h"].dtype)}


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


def _at(s, name):
    return s[name].data_ptr() if name in s else None


def _own(s):
    p, rt = _reactor()
    case = s["case"]
    kind = case["kind"]
    dtype = p.DTYPE_BF16 if case["type"] == BF16 else p.DTYPE_F32
    if kind in ("pack", "product"):
        n, k = case["n"], case["k"]
        matrix = p.w4_matrix(s["packed"].data_ptr(), n, k, case["group"])
        if kind == "pack":
            rt.w4_pack_device(matrix, s["w"].data_ptr(), k, dtype)
            rt.w4_unpack_device(matrix, s["out"].data_ptr(), k, dtype)
        else:
            rt.gemm_w4_device(matrix, s["x"].data_ptr(), s["out"].data_ptr(), case["m"], k, n, dtype)
        return s["out"]
    if kind == "mixture":
        gate, up, down = (p.w4_matrix(s[name].data_ptr(), n, k, case["group"], case["experts"])
                          for name, (n, k) in _expert_shapes(case).items())
        rt.moe_w4_device(gate, up, down, s["router"].data_ptr(), s["x"].data_ptr(), s["out"].data_ptr(), case["tokens"],
                         case["top_k"], case["hidden"], case["hidden"], dtype,
                         activation=p.MOE_SILU if case["act"] == SILU else p.MOE_GELU_TANH,
                         renormalise=case["renormalise"], dexperts=s["chosen"].data_ptr(),
                         dweights=s["weights"].data_ptr())
        return {"out": s["out"], "chosen": s["chosen"], "weights": s["weights"]}
    if kind == "rope":
        q, k, dim = case["q_heads"], case["k_heads"], case["dim"]
        rt.rope_device(s["positions"].data_ptr(), s["turns"].data_ptr(), case["rows"], dim, case["rotary"],
                       p.ROPE_HALF if case["layout"] == "half" else p.ROPE_PAIRS, dtype, magnitude=s["magnitude"],
                       q=(s["q"].data_ptr(), s["q_out"].data_ptr(), q, q * dim, q * dim),
                       k=(s["k"].data_ptr(), s["k_out"].data_ptr(), k, k * dim, k * dim))
        return {"q": s["q_out"], "k": s["k_out"]}
    rt.residual_norm_device(s["h"].data_ptr(), s["h_out"].data_ptr(), s["out"].data_ptr(), case["rows"], case["width"],
                            dtype, dy=s["y"].data_ptr(), dpost=_at(s, "post"), dgate=_at(s, "gate"), gate_tanh=True,
                            dpre=s["pre"].data_ptr(), dscale=_at(s, "scale"), dshift=_at(s, "shift"),
                            rows_per_vector=case["per"], residual_scale=case["residual_scale"], eps=EPS)
    return {"h": s["h_out"], "out": s["out"]}


_PLAIN = {"pack": _plain_pack, "product": _plain_product, "mixture": _plain_mixture, "rope": _plain_rope,
          "norm": _plain_norm}


def run(s):
    return _own(s) if own else _PLAIN[s["case"]["kind"]](s)


def work(case) -> dict:
    size = 4 if case["type"] == F32 else 2
    kind = case["kind"]
    held = lambda n, k: n * k // 2 + 2 * n * -(-k // case["group"])  # noqa: E731
    if kind == "pack":
        n, k = case["n"], case["k"]
        # weights in, packed out, packed in, weights out
        return {"bytes": 2 * n * k * size + 2 * held(n, k), "flops": 16 * n * k}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": held(n, k) + size * m * (n + k), "flops": 2 * m * n * k}
    if kind == "mixture":
        tokens, hidden, inner, experts = case["tokens"], case["hidden"], case["inner"], case["experts"]
        pairs = tokens * case["top_k"]
        # As many experts as even choices reach.
        reached = experts * (1.0 - (1.0 - case["top_k"] / experts) ** tokens)
        weights = 2 * held(inner, hidden) + held(hidden, inner)
        return {"bytes": int(reached * weights) + 4 * experts * hidden + 2 * size * tokens * hidden + 8 * pairs,
                "flops": 6 * pairs * hidden * inner + 2 * tokens * experts * hidden}
    if kind == "rope":
        values = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": 2 * size * values + 4 * case["rows"], "flops": 3 * values}
    values, vectors = case["rows"] * case["width"], -(-case["rows"] // case["per"]) * case["width"]
    shared = int(case["gate"]) + 2 * int(case["modulate"])
    return {"bytes": size * (4 * values + shared * vectors) + 8 * case["width"], "flops": 12 * values}


# ------------------------------------------------------- the same in 64 bits
def _to32(x):
    """One rounding to 32 bits, as the definitions ask of a quotient."""
    return x.to(torch.float32).to(torch.float64)


def _exact_values(w, group):
    """What the weights w are held as, value by value from the definition."""
    n, k = w.shape
    g = torch.nn.functional.pad(w.double(), (0, -k % group)).reshape(n, -1, group)
    # mantissa in [1/2, 1): six significant bits are 64ths of the power of two above
    mantissa, exponent = torch.frexp(_to32(g.abs().max(-1)[0] / 6.0))
    step = torch.ldexp(torch.ceil(mantissa * 64.0) / 64.0, exponent)[..., None]
    y = torch.where(step > 0.0, _to32(g / step), 0.0)
    # The distance between neighbours doubles at 2 and at 4, and an even multiple of it is an even code.
    unit = torch.where(y.abs() < 2.0, 0.5, torch.where(y.abs() < 4.0, 1.0, 2.0))
    return (step * (torch.round(y / unit) * unit)).reshape(n, -1)[:, :k]


def _exact_mixture(case, seed, x):
    rows = x["x"].double()
    logits = (rows[:, None, :] * x["router"].double()[None]).sum(-1)
    # The place of an expert: how many are before it.
    lower = torch.ones(case["experts"], case["experts"], dtype=torch.bool, device="cuda").tril(-1)
    ahead = (logits[:, None, :] > logits[:, :, None]) | ((logits[:, None, :] == logits[:, :, None]) & lower)
    place = ahead.sum(-1)
    p = torch.softmax(logits, -1)
    taken = place < case["top_k"]
    if case["renormalise"]:
        p = p / torch.where(taken, p, 0.0).sum(-1, keepdim=True)
    out = torch.zeros_like(rows)
    for e, w in enumerate(_experts(case, seed)):
        token = taken[:, e].nonzero()[:, 0]
        if len(token) == 0:
            continue
        w = {name: _exact_values(t, case["group"]).t().contiguous() for name, t in w.items()}
        g = rows[token] @ w["gate"]
        if case["act"] == SILU:
            g = g * torch.sigmoid(g)
        else:
            g = g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
        out[token] += p[token, e, None] * ((g * (rows[token] @ w["up"])) @ w["down"])
    chosen = torch.argsort(place, -1)[:, :case["top_k"]]
    return {"out": out, "chosen": chosen.int(), "weights": p.gather(1, chosen)}


def _exact_rope(case, x):
    frequencies, magnitude = _frequencies(case)
    turned = torch.polar(torch.full((case["rows"], case["rotary"] // 2), magnitude, dtype=torch.float64, device="cuda"),
                         x["positions"].double()[:, None] * frequencies.to("cuda"))[:, None]
    out = {}
    for name in ("q", "k"):
        y = x[name].double()
        front = y[..., :case["rotary"]]
        if case["layout"] == "half":
            z = torch.complex(*front.unflatten(-1, (2, -1)).unbind(-2)) * turned
            front = torch.cat((z.real, z.imag), -1)
        else:
            front = torch.view_as_real(torch.view_as_complex(front.unflatten(-1, (-1, 2)).contiguous()) * turned).flatten(-2)
        out[name] = torch.cat((front, y[..., case["rotary"]:]), -1)
    return out


def _exact_norm(case, x):
    x = {name: t.double() for name, t in x.items()}
    shared = lambda name: x[name].repeat_interleave(case["per"], 0)[:case["rows"]]  # noqa: E731
    size = lambda t: (t.square().sum(-1, keepdim=True) / case["width"] + EPS).sqrt()  # noqa: E731
    y = x["y"]
    if case["post"]:
        y = y / size(y) * x["post"]
    if case["gate"]:
        y = y * shared("gate").tanh()
    h = x["h"] + case["residual_scale"] * y
    out = h / size(h) * x["pre"]
    if case["modulate"]:
        out = out + out * shared("scale") + shared("shift")
    return {"h": h, "out": out}


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "pack":
        return _exact_values(x["w"], case["group"])
    if kind == "product":
        return x["x"].double() @ _exact_values(x["w"], case["group"]).t().contiguous()
    if kind == "mixture":
        return _exact_mixture(case, seed, x)
    return _exact_rope(case, x) if kind == "rope" else _exact_norm(case, x)
