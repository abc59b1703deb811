"""The quantised serving operators as they are measured: cases, inputs, one pass, its work, its exact outputs.

Four operators: the residual add with RMSNorm and 8-bit rows out (``norm``), the 8-bit integer product with a
scale per token and per channel (``linear``), the 4-bit ring cache written and read back (``cache``) and one
decoding token's attention over it (``attend``). ``own`` selects the package's entry points; otherwise the same
values come from elementary torch operations in 32 bits.

Formats. 8-bit rows: codes in [-127, 127] and one float32 scale per row. 4-bit ring: per (row, key head, slot) the
channels fall in groups of 32 (16 where the head dimension is not a multiple of 32); a group keeps ``lo`` (its minimum
rounded down to bf16) and ``step`` ((max - lo) / 15 rounded up to bf16) and a code 0..15 per channel, two codes a
byte: (x - lo) / step rounded to the nearest whole number, ties to even. The channels' order in a slot's bytes is
given by ``key_order`` and ``value_order``. ``pos`` holds each slot's position, -1 where nothing was written; a token
at position p lives in slot p % window.
"""

import math

import torch

own = False

FLOOR, EPS = 1e-3, 1e-6
TINY_ROW = 1e-35  # rows below this are zero
TINY_RANGE = 2.0**-100  # groups whose range is below this are flat
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
SLOT_TILE = 64  # a ring's slots are allocated in tiles of 64


def listed():
    return [
        # a decode step's norm: 64 streams of the width-512 model, float32 residual stream plus a bf16 sublayer output
        {"name": "norm decode 64x512", "op": "norm", "rows": 64, "width": 512, "r": "bf16"},
        # the norms of one training-size batch run as prefill (16 x 2048 tokens)
        {"name": "norm prefill 32768x512", "op": "norm", "rows": 32768, "width": 512, "r": "bf16"},
        # a wide model's ragged prefill: odd row count, a width that fills no power of two, float32 sublayer output
        {"name": "norm wide 7001x5000", "op": "norm", "rows": 7001, "width": 5000, "r": "f32"},
        # a decode step's recurrent projections as one product: 64 streams, q, k, v and 8 write strengths (3 x 512 + 8)
        {"name": "linear decode 64x512x1544", "op": "linear", "m": 64, "k": 512, "n": 1544, "out": "bf16"},
        # one stream of a wide model: every weight byte is read for a single token
        {"name": "linear one 1x4096x8192", "op": "linear", "m": 1, "k": 4096, "n": 8192, "out": "bf16"},
        # a ragged batch of prompts, sizes no tile divides, float32 out
        {"name": "linear odd 777x1040x2001", "op": "linear", "m": 777, "k": 1040, "n": 2001, "out": "f32"},
        # prefill of a wide model's feed-forward block: the product that the tensor cores bound
        {"name": "linear prefill 8192x4096x8192", "op": "linear", "m": 8192, "k": 4096, "n": 8192, "out": "bf16"},
        # a prefill chunk entering the decode rings: 64 streams x 2048 tokens, windows of 512, read back for the next chunk
        {"name": "cache chunk 64x2048 w512", "op": "cache", "b": 64, "n": 2048, "hkv": 2, "dk": 64, "window": 512, "t": "bf16"},
        # long prompts into long rings, wide heads, an odd prompt length
        {"name": "cache long 4x32701 w32768", "op": "cache", "b": 4, "n": 32701, "hkv": 8, "dk": 128, "window": 32768, "t": "bf16"},
        # a decode step's attention: 64 streams, 8 query heads over 2 key heads, full windows of 512
        {"name": "attend decode 64 w512", "op": "attend", "b": 64, "h": 8, "hkv": 2, "dk": 64, "window": 512, "held": 512,
         "ragged": False, "t": "bf16"},
        # long contexts of different lengths: streams hold from an eighth of 49999 positions up to all of them
        {"name": "attend long 8 ragged", "op": "attend", "b": 8, "h": 32, "hkv": 8, "dk": 128, "window": 65536, "held": 49999,
         "ragged": True, "t": "bf16"},
        # one stream over a long window in float32, the only work on the card
        {"name": "attend one f32", "op": "attend", "b": 1, "h": 8, "hkv": 2, "dk": 64, "window": 131072, "held": 100003,
         "ragged": False, "t": "f32"},
    ]  # fmt: skip


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "cache", "attend"])
    if op == "norm":
        width = 4 * _spread(rng, 8, 2000)
        rows = _spread(rng, 1, 35_000_000 // width)
        return {"op": op, "rows": rows, "width": width, "r": rng.choice(["bf16", "f16", "f32"])}
    if op == "linear":
        k, n = 16 * _spread(rng, 4, 512), _spread(rng, 16, 8192)
        m = _spread(rng, 1, min(16384, 8192 * 4096 * 8192 // (k * n)))
        return {"op": op, "m": m, "k": k, "n": n, "out": rng.choice(["bf16", "f16", "f32"])}
    dk = rng.choice([16, 32, 48, 64, 64, 96, 128, 128])
    hkv = rng.choice([1, 2, 3, 4, 8])
    if op == "cache":
        most = 4 * 32701 * 8 * 128 // (hkv * dk)
        b = rng.choice([1, 2, 5, 16, 64])
        n = _spread(rng, 1, min(40000, most // b))
        window = _spread(rng, 16, min(40000, most // b))
        return {"op": op, "b": b, "n": n, "hkv": hkv, "dk": dk, "window": window, "t": rng.choice(["bf16", "f16", "f32"])}
    b = rng.choice([1, 2, 7, 16, 64])
    window = _spread(rng, 16, min(131072, 4 * 49999 * 8 * 128 // (hkv * dk * b)))
    return {"op": op, "b": b, "h": hkv * rng.choice([1, 2, 3, 4, 5, 8]), "hkv": hkv, "dk": dk, "window": window,
            "held": _spread(rng, 1, window), "ragged": rng.random() < 0.5, "t": rng.choice(["bf16", "f16", "f32"])}  # fmt: skip


def lengths(case):
    """Positions each stream holds before its token, the token's position being the stream's length."""
    b, held = case["b"], case["held"]
    return [max(1, held * (i + 1) // b) if case["ragged"] else held for i in range(b)]


def group_size(dk):
    return 32 if dk % 32 == 0 else 16


def slots_of(window):
    return -(-window // SLOT_TILE) * SLOT_TILE


def work(case):
    op = case["op"]
    if op == "norm":
        n, w = case["rows"], case["width"]
        return {"bytes": n * w * (4 + SIZE[case["r"]] + 4 + 1) + 4 * (n + w), "flops": 8 * n * w}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k + n * k + m * n * SIZE[case["out"]] + 4 * (m + n), "flops": 2 * m * k * n}
    row = case["dk"] // 2 + 4 * (case["dk"] // group_size(case["dk"]))  # bytes of one slot's keys or values
    if op == "cache":
        kept, heads, e = min(case["n"], case["window"]), case["b"] * case["hkv"], SIZE[case["t"]]
        vals = 2 * heads * kept * case["dk"]
        return {"bytes": 2 * vals * e + 4 * heads * kept * row + 25 * case["b"] * kept, "flops": 10 * vals}
    seen = sum(min(x + 1, case["window"]) for x in lengths(case))
    return {"bytes": seen * (2 * case["hkv"] * row + 8) + 2 * case["b"] * case["h"] * case["dk"] * SIZE[case["t"]],
            "flops": 4 * seen * case["h"] * case["dk"]}  # fmt: skip


# ---- inputs -----------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "norm":
        n, w = case["rows"], case["width"]
        # a residual stream: rows of different size, a few channels much larger than the rest
        gain = 1 + 0.2 * _normal(g, w)
        x = _normal(g, n, w) * torch.exp(0.5 * _normal(g, n, 1)) * torch.exp(0.7 * _normal(g, w))
        return {"case": case, "x": x, "r": _normal(g, n, w, dtype=TYPES[case["r"]]), "gain": gain}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        xq, xs = plain_rows(_normal(g, m, k) * torch.exp(0.7 * _normal(g, k)))
        wq, ws = plain_rows(_normal(g, n, k) / math.sqrt(k))
        return {"case": case, "xq": xq, "xs": xs, "wq": wq, "ws": ws}
    b, hkv, dk, window = case["b"], case["hkv"], case["dk"], case["window"]
    dtype, slots = TYPES[case["t"]], slots_of(window)
    # keys have channels with an offset of their own, values do not
    shift = 2 * _normal(g, hkv, dk) * (torch.rand(hkv, dk, device="cuda", generator=g) < 0.1)
    ng = dk // group_size(dk)
    ring = {
        "k_codes": torch.zeros(b, hkv, slots, dk // 2, dtype=torch.uint8, device="cuda"),
        "k_params": torch.zeros(b, hkv, slots, ng, 2, dtype=torch.bfloat16, device="cuda"),
        "v_codes": torch.zeros(b, hkv, slots, dk // 2, dtype=torch.uint8, device="cuda"),
        "v_params": torch.zeros(b, hkv, slots, ng, 2, dtype=torch.bfloat16, device="cuda"),
        "pos": torch.full((b, slots), -1, dtype=torch.long, device="cuda"),
    }
    if case["op"] == "cache":
        n = case["n"]
        first = int(torch.randint(0, 1000, (1,), device="cuda", generator=g))
        pos = torch.arange(first, first + n, device="cuda").expand(b, n).contiguous()
        kept = min(n, window)
        return {"case": case, "ring": ring, "k": (_normal(g, b, n, hkv, dk) + shift).to(dtype),
                "v": _normal(g, b, n, hkv, dk, dtype=dtype), "pos": pos, "back": pos[:, n - kept :].contiguous()}  # fmt: skip
    at = torch.tensor(lengths(case), device="cuda")[:, None]  # [b, 1]: the token's position
    slot = torch.arange(slots, device="cuda")[None, :]
    last = at - 1  # slot s holds the newest position <= last that is s modulo the window
    p = last - (last - slot) % window
    ring["pos"] = torch.where((slot < window) & (p >= 0), p, -1)
    for name, off in (("k", shift[:, None, :]), ("v", 0.0)):
        for i in range(b):
            x = _normal(g, hkv, slots, dk) + off
            codes, params = plain_groups(x)
            ring[name + "_codes"][i] = plain_pack(codes, name)
            ring[name + "_params"][i] = params
    return {"case": case, "ring": ring, "q": _normal(g, b, 1, case["h"], dk, dtype=dtype),
            "k": (_normal(g, b, 1, hkv, dk) + shift).to(dtype), "v": _normal(g, b, 1, hkv, dk, dtype=dtype),
            "pos": at.contiguous()}  # fmt: skip


# ---- the plain forms --------------------------------------------------------------------------------------


def plain_rows(y):
    """8-bit codes and scales of float32 rows."""
    amax = y.abs().amax(-1, keepdim=True)
    live = torch.isfinite(amax) & (amax >= TINY_ROW)
    most = torch.full_like(amax, 127.0)  # tensors, so that both quotients are divisions
    inverse = torch.where(live, most / amax, 0.0)
    scale = torch.where(live, amax / most, torch.where(torch.isfinite(amax), 0.0, math.nan))
    return torch.where(live, torch.round(y * inverse), 0.0).to(torch.int8), scale[..., 0]


def _cut(x):
    """Float32 with the low 16 bits cleared (bf16 towards zero), and whether bits were lost."""
    bits = x.contiguous().view(torch.int32)
    return (bits & -65536), (bits & 65535) != 0


def plain_groups(x):
    """4-bit codes ``[..., dk]`` and (step, lo) pairs ``[..., groups, 2]`` of float32 ``x [..., dk]``."""
    dk = x.shape[-1]
    xg = x.unflatten(-1, (dk // group_size(dk), group_size(dk)))
    low, high = xg.amin(-1), xg.amax(-1)
    bits, lost = _cut(low)
    lo = torch.where(lost & (low < 0), bits + 65536, bits).view(torch.float32)
    span = high - lo
    bits, lost = _cut(span / torch.full_like(span, 15.0))
    step = torch.where(lost, bits + 65536, bits).view(torch.float32)
    flat = span < TINY_RANGE
    bad = ~(torch.isfinite(step) & torch.isfinite(lo))
    step = torch.where(bad, math.nan, torch.where(flat, 0.0, step))
    lo = torch.where(bad, math.nan, lo)
    codes = torch.round((xg - lo[..., None]) / step[..., None]).clamp(max=15.0)
    codes = torch.where((flat | bad)[..., None], 0.0, codes)
    return codes.to(torch.uint8).flatten(-2), torch.stack([step, lo], -1).to(torch.bfloat16)


def plain_pack(codes, which):
    """Bytes ``[..., dk/2]`` of codes ``[..., dk]`` in the cache's order (first of a pair in the low half)."""
    dk = codes.shape[-1]
    if which == "k":
        x = codes.unflatten(-1, (dk // group_size(dk), 4, group_size(dk) // 4)).transpose(-3, -2)
    else:
        x = codes.unflatten(-1, (dk // 16, 8, 2)).transpose(-3, -2)
    x = x.flatten(-3).unflatten(-1, (dk // 2, 2))
    return x[..., 0] | (x[..., 1] << 4)


def plain_values(data, params, which):
    """Float32 values ``[..., dk]`` of a cache's bytes and parameters."""
    dk = 2 * data.shape[-1]
    x = torch.stack([data & 15, data >> 4], -1).flatten(-2)
    if which == "k":
        x = x.unflatten(-1, (4, dk // group_size(dk), group_size(dk) // 4)).transpose(-3, -2).flatten(-3)
    else:
        x = x.unflatten(-1, (8, dk // 16, 2)).transpose(-3, -2).flatten(-3)
    x = x.unflatten(-1, (dk // group_size(dk), group_size(dk))).float()
    p = params.float()
    return (p[..., 1:] + x * p[..., :1]).flatten(-2)


def _plain_norm(s):
    x = s["x"] + s["r"].float()
    c = x.abs().amax(-1, keepdim=True).clamp(min=FLOOR)
    z = x / c
    y = z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS / (c * c)) * s["gain"]
    q, scale = plain_rows(y)
    return {"sum": x, "values": (q.float() * scale[:, None]).to(torch.bfloat16), "scale": scale}


def _plain_linear(s):
    acc = s["xq"].float() @ s["wq"].float().T
    return (acc * s["xs"][:, None] * s["ws"]).to(TYPES[s["case"]["out"]])


def _plain_write(s, window):
    ring, n = s["ring"], s["pos"].shape[1]
    kept = min(n, window)
    pos = s["pos"][:, n - kept :]
    slot, row = pos % window, torch.arange(pos.shape[0], device=pos.device)[:, None]
    for name in ("k", "v"):
        codes, params = plain_groups(s[name][:, n - kept :].float())
        ring[name + "_codes"][row, :, slot] = plain_pack(codes, name)
        ring[name + "_params"][row, :, slot] = params
    ring["pos"][row, slot] = pos


def _plain_read(ring, pos, window, dtype):
    slot, row = pos % window, torch.arange(pos.shape[0], device=pos.device)[:, None]
    held = ring["pos"][row, slot] == pos
    k = plain_values(ring["k_codes"][row, :, slot], ring["k_params"][row, :, slot], "k")
    v = plain_values(ring["v_codes"][row, :, slot], ring["v_params"][row, :, slot], "v")
    keep = held[:, :, None, None]
    return torch.where(keep, k, 0.0).to(dtype), torch.where(keep, v, 0.0).to(dtype), held


def _plain_attend(s):
    case, ring, pos = s["case"], s["ring"], s["pos"]
    b, hkv, dk, window = case["b"], case["hkv"], case["dk"], case["window"]
    _plain_write(s, window)
    k, v = (plain_values(ring[n + "_codes"], ring[n + "_params"], n) for n in ("k", "v"))
    q = s["q"].float().view(b, hkv, -1, dk)
    seen = (ring["pos"] >= 0) & (ring["pos"] <= pos) & (ring["pos"] > pos - window)
    scores = (q @ k.transpose(-1, -2)) / math.sqrt(dk)
    scores = torch.where(seen[:, None, None, :], scores, -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (w @ v) / w.sum(-1, keepdim=True)
    k1, v1, _ = _plain_read(ring, pos, window, s["k"].dtype)
    return {"o": o.reshape(s["q"].shape).to(s["q"].dtype), "k": k1, "v": v1}


def _plain_cache(s):
    window = s["case"]["window"]
    _plain_write(s, window)
    k, v, held = _plain_read(s["ring"], s["back"], window, s["k"].dtype)
    return {"k": k, "v": v, "held": held}


def _own(s):
    case = s["case"]
    if case["op"] == "norm":
        from vesper_b200.kernels.q8 import add_rms_norm_q8, dequantize_rows_q8

        total, q, scale = add_rms_norm_q8(s["x"], s["r"], s["gain"], FLOOR, EPS)
        return {"sum": total, "values": dequantize_rows_q8(q, scale, torch.bfloat16), "scale": scale}
    if case["op"] == "linear":
        from vesper_b200.kernels.q8 import linear_q8

        return linear_q8(s["xq"], s["xs"], s["wq"], s["ws"], TYPES[case["out"]])
    from vesper_b200.kernels.q4_cache import Q4RingKVCache, q4_attend_, q4_read, q4_write_

    ring = Q4RingKVCache(**s["ring"], window=case["window"])
    if case["op"] == "cache":
        q4_write_(ring, s["k"], s["v"], s["pos"])
        k, v, held = q4_read(ring, s["back"], s["k"].dtype)
        return {"k": k, "v": v, "held": held}
    o = q4_attend_(s["q"], s["k"], s["v"], s["pos"], ring)
    k, v, _ = q4_read(ring, s["pos"], s["k"].dtype)  # what the ring now holds of the token
    return {"o": o, "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"norm": _plain_norm, "linear": _plain_linear, "cache": _plain_cache, "attend": _plain_attend}[op](state)


# ---- exact outputs in 64 bits, from the definitions ----------------------------------------------------------


def _exact_round(y, down):
    """The nearest bf16 not above (``down``) or not below ``y`` (float64)."""
    near = y.to(torch.bfloat16).double()
    mantissa, exponent = torch.frexp(near)
    ulp = torch.ldexp(torch.ones_like(mantissa), exponent - 8)
    # one bf16 step towards zero from a power of two is half as long
    shrink = torch.where(mantissa.abs() == 0.5, ulp / 2, ulp)
    if down:
        return torch.where(near > y, near - torch.where(near > 0, shrink, ulp), near)
    return torch.where(near < y, near + torch.where(near < 0, shrink, ulp), near)


def _exact_stored(x):
    """The values that a 4-bit group keeps of ``x [..., dk]`` (float64)."""
    size = group_size(x.shape[-1])
    g = x.reshape(*x.shape[:-1], -1, size)
    lo = _exact_round(g.min(-1, keepdim=True).values, True)
    span = g.max(-1, keepdim=True).values - lo
    step = _exact_round(span / 15, False)
    flat = span < TINY_RANGE
    code = torch.where(flat, 0.0, ((g - lo) / torch.where(flat, 1.0, step)).round().clamp(max=15))
    return (lo + code * torch.where(flat, 0.0, step)).reshape(x.shape)


def key_order(dk):
    """The channel at each place of a slot's key codes."""
    size = group_size(dk)
    return [g * size + t * (size // 4) + i for t in range(4) for g in range(dk // size) for i in range(size // 4)]


def value_order(dk):
    """The channel at each place of a slot's value codes."""
    return [16 * i + 2 * g + r for g in range(8) for i in range(dk // 16) for r in range(2)]


def _exact_decode(data, params, order):
    size = group_size(len(order))
    out = torch.empty(*data.shape[:-1], len(order), dtype=torch.float64, device=data.device)
    for place, channel in enumerate(order):
        code = (data[..., place // 2].long() >> (4 * (place % 2))) % 16
        p = params[..., channel // size, :].double()
        out[..., channel] = p[..., 1] + code * p[..., 0]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double() + s["r"].double()
        y = x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * s["gain"].double()
        scale = y.abs().max(1).values / 127
        return {"sum": x, "values": torch.round(y / scale[:, None]) * scale[:, None], "scale": scale}
    if case["op"] == "linear":
        return torch.matmul(s["xq"].double() * s["xs"].double()[:, None], s["wq"].double().T) * s["ws"].double()
    if case["op"] == "cache":
        kept = s["back"].shape[1]
        return {"k": _exact_stored(s["k"][:, -kept:].double()), "v": _exact_stored(s["v"][:, -kept:].double()), "held": None}
    b, hkv, dk, window = case["b"], case["hkv"], case["dk"], case["window"]
    k1, v1 = _exact_stored(s["k"].double()), _exact_stored(s["v"].double())
    out = torch.empty(b, hkv, case["h"] // hkv, dk, dtype=torch.float64, device="cuda")
    for i in range(b):
        p = int(s["pos"][i, 0])
        here = s["ring"]["pos"][i]
        at = torch.nonzero((here >= 0) & (here > p - window) & (here < p))[:, 0]
        k, v = (_exact_decode(s["ring"][n + "_codes"][i][:, at], s["ring"][n + "_params"][i][:, at], order)
                for n, order in (("k", key_order(dk)), ("v", value_order(dk))))  # fmt: skip
        k, v = torch.cat([k, k1[i].transpose(0, 1)], 1), torch.cat([v, v1[i].transpose(0, 1)], 1)
        q = s["q"][i, 0].double().view(hkv, -1, dk)
        out[i] = torch.softmax(torch.einsum("hgd,hld->hgl", q, k) * dk**-0.5, -1) @ v
    return {"o": out.view(b, 1, case["h"], dk), "k": k1, "v": v1}
