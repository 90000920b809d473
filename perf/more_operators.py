"""Performance cases of 4-bit numbers (blocks of 32 e2m1 values under a power of two) and of the paged memory that holds
them.

Four kinds of work:

    append   kv_append: a step's or a chunk's queries and keys turned by their positions, keys and values into their pages
    attend   paged_attention of each sequence's new tokens over pages of 4 bits
    pack     mx_pack of rows, then mx_unpack of what they became
    linear   mx_linear: a linear layer with 4-bit weights on rows that it packs

listed() holds sizes that an image encoder, a video's memory bank and a server's decoding have; draw() gives others of the
same ranges.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
E4M3_MAX, E2M1_MAX, BLOCK = 448.0, 6.0, 32


def _hip():
    if "sam_hip" not in sys.modules:  # a program imports it once
        sys.path.insert(0, os.path.abspath("sam-rs_amd"))
        import sam_hip  # noqa: F401
    return sys.modules["sam_hip"]


def listed():
    return [
        # A decoding step of 32 sequences into 4 bits, each with a short history that is read back. Latency.
        {"name": "append_steps_fp4_bf16", "kind": "append", "dtype": "bf16", "held": "e2m1", "b": 32, "chunk": 1, "len": 40,
         "ragged": 0.8, "hkv": 8, "g": 4, "d": 128, "page": 16, "pairs": "halves", "sections": "64", "pos": False},
        # A frame of 4096 queries and keys at (time, row, column) enters a video's memory in 8 bits, which is read back.
        {"name": "append_frame_fp8_f16", "kind": "append", "dtype": "f16", "held": "e4m3", "b": 1, "chunk": 4096,
         "len": 28736, "ragged": 0.0, "hkv": 1, "g": 1, "d": 256, "page": 64, "pairs": "adjacent", "sections": "32,48,48",
         "pos": True},
        # Five prompts of different lengths into 16-bit pages, 16 query and 4 key heads of 128, three quarters turned.
        {"name": "append_prompts_bf16", "kind": "append", "dtype": "bf16", "held": "own", "b": 5, "chunk": 4001,
         "len": 4500, "ragged": 0.8, "hkv": 4, "g": 4, "d": 128, "page": 16, "pairs": "halves", "sections": "48", "pos": False},
        # One token over a short history, 8 heads of 64: latency.
        {"name": "attend_token_f16", "kind": "attend", "dtype": "f16", "b": 1, "chunk": 1, "len": 577, "ragged": 0.0,
         "hkv": 8, "g": 1, "d": 64, "page": 16, "causal": True},
        # A server's decoding step: 32 sequences of up to 8192 tokens, 32 query and 8 key heads of 128.
        {"name": "attend_steps_bf16", "kind": "attend", "dtype": "bf16", "b": 32, "chunk": 1, "len": 8192, "ragged": 0.9,
         "hkv": 8, "g": 4, "d": 128, "page": 16, "causal": True},
        # One token over a long history, 16 query and 2 key heads of 128.
        {"name": "attend_long_f16", "kind": "attend", "dtype": "f16", "b": 1, "chunk": 1, "len": 131072, "ragged": 0.0,
         "hkv": 2, "g": 8, "d": 128, "page": 64, "causal": True},
        # SAM 2.1's memory attention, cross: a frame's 4096 queries over 7 frames and 64 pointer tokens.
        {"name": "attend_memory_f16", "kind": "attend", "dtype": "f16", "b": 1, "chunk": 4096, "len": 28736, "ragged": 0.0,
         "hkv": 1, "g": 1, "d": 256, "page": 64, "causal": False},
        # One window's activations of ViT-H in 32 bits, 196 tokens.
        {"name": "pack_window_f32", "kind": "pack", "dtype": "f32", "m": 196, "k": 1280},
        # The MLP's activations of eight images of ViT-H.
        {"name": "pack_images_f16", "kind": "pack", "dtype": "f16", "m": 32768, "k": 5120},
        # The MLP's second layer of ViT-H on seven tokens. Latency and the weights' bytes.
        {"name": "linear_few_f32", "kind": "linear", "dtype": "f32", "m": 7, "n": 1280, "k": 5120, "bias": True, "gelu": False},
        # The MLP's first layer of ViT-H on one image.
        {"name": "linear_image_f16", "kind": "linear", "dtype": "f16", "m": 4096, "n": 5120, "k": 1280, "bias": True,
         "gelu": True},
        # The MLP's second layer of ViT-L on a batch of images whose last one is cut short.
        {"name": "linear_batch_bf16", "kind": "linear", "dtype": "bf16", "m": 16001, "n": 1024, "k": 4096, "bias": False,
         "gelu": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "pack", "linear", "linear"])
    dtype = rng.choice(["f16", "f16", "f16", "bf16", "bf16", "bf16", "f32"])
    if kind == "pack":
        return {"kind": kind, "dtype": dtype, "m": _log(rng, 1, 65536), "k": BLOCK * _log(rng, 1, 256)}
    if kind == "linear":
        return {"kind": kind, "dtype": dtype, "m": _log(rng, 1, 16384), "n": _log(rng, 1, 8192),
                "k": BLOCK * _log(rng, 1, 256), "bias": rng.random() < 0.5, "gelu": rng.random() < 0.3}
    b = _log(rng, 1, 64)
    length = _log(rng, 1, 65536)
    case = {"kind": kind, "dtype": dtype, "b": b, "chunk": min(length, rng.choice([1, 1, _log(rng, 1, 4096)])),
            "len": length, "ragged": rng.choice([0.0, 0.5, 0.9]), "hkv": _log(rng, 1, 16),
            "g": rng.choice([1, 1, 2, 3, 4, 6, 8]), "d": rng.choice([32, 64, 96, 128, 160, 256]),
            "page": rng.choice([8, 16, 24, 32, 64, 100, 128, 256])}
    if kind == "attend":
        case["causal"] = rng.random() < 0.6
        return case
    case["held"] = rng.choice(["own", "e4m3", "e2m1"])
    if case["held"] != "e2m1":
        case["d"] = rng.choice([64, 72, 80, 96, 128, 256])
    half = case["d"] // 2
    rows = rng.randint(1, half // 2)
    case["pos"] = rng.random() < 0.5
    turned = rng.choice([half, half, rng.randint(rows + 1, half)])
    case["sections"] = "%d,%d" % (rows, turned - rows) if case["pos"] else str(turned)
    case["pairs"] = rng.choice(["adjacent", "halves"])
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / (1e14 if case["dtype"] == "f32" else 1e15))


def _room(case):
    """Bytes that the plain form holds at most: the keys and values and the scores of a padded batch in 32 bits."""
    if case["kind"] in ("pack", "linear"):
        return 0
    n = 4 * 4 * case["b"] * case["hkv"] * case["len"] * case["d"]
    if case["kind"] == "attend":
        n += 3 * 4 * case["b"] * case["hkv"] * case["g"] * case["chunk"] * case["len"]
    else:
        n += 4 * 8 * case["b"] * case["chunk"] * case["hkv"] * (case["g"] + 2) * case["d"]
    return n


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _drawn(rng)
        if _cost(case) <= most and _room(case) <= 16e9:
            return case


# ------------------------------------------------------------------------------------------------- inputs


def _spread(b, n, most, ragged):
    """Lengths of n sequences: the longest `most`, the others down to (1 - ragged) of it, in a fixed irregular order."""
    return max(1, int(round(most * (1.0 - ragged * ((b * 0.6180339887498949) % 1.0)))))


def _lengths(case):
    chunks = [_spread(i + 3 if i else 0, case["b"], case["chunk"], case["ragged"]) for i in range(case["b"])]
    lens = [max(c, _spread(i, case["b"], case["len"], case["ragged"])) for i, c in enumerate(chunks)]
    return chunks, lens


def _power(s, dtype=torch.float32):
    """2^s exactly, for whole s of a normal result."""
    if dtype == torch.float64:
        return ((s.long() + 1023) << 52).view(torch.float64)
    return ((s + 127).to(torch.int32) << 23).view(torch.float32)


def _least(top, lift):
    """The least s within +-126 with top <= 1.75 * 2^(s + 8) (lift 9: e4m3's 448) or 1.5 * 2^(s + 2) (lift 3: e2m1's 6)."""
    m, e = torch.frexp(top)
    return torch.where(top > 0, e - lift + (m > (0.875 if lift == 9 else 0.75)).to(e.dtype), 0).clamp(-126, 126)


def _mx(x):
    """e2m1 values (over their scales) of x's blocks of 32 and the biased exponents of those; a block with a value that is not
    finite has 255, and zeros."""
    y = x.unflatten(-1, (-1, BLOCK))
    fine = torch.isfinite(y).all(-1)
    y = torch.where(fine[..., None], y, 0.0)
    s = _least(y.abs().amax(-1), 3)
    y = y * _power(-s, y.dtype)[..., None]
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).to(y.dtype)
    return torch.round(y / step) * step, torch.where(fine, s + 127, 255).to(torch.uint8)


def _mx_codes(v):
    """Codes of e2m1 values, two to a byte, the even column's in the low half."""
    v = v.flatten(-2)
    a = v.abs()
    c = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4


def _mx_values(codes, scale, dtype=torch.float32):
    """What codes and scales stand for."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device, dtype=dtype)
    grid = torch.cat([grid, -grid])
    two = torch.where(scale == 255, float("nan"), _power(scale.int().clamp(max=254) - 127, dtype))
    x = grid[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    return (x.unflatten(-1, (-1, BLOCK)) * two[..., None]).flatten(-2)


def _e4m3(x):
    """e4m3 codes of rows and the biased exponents of their scales, the powers of two that bring a row's largest
    value to 448 at most and as near to it as they can."""
    s = _least(x.abs().amax(-1), 9)
    return (x * _power(-s, x.dtype)[..., None]).float().to(torch.float8_e4m3fn), (s + 127).to(torch.uint8)


def _pool(held, dtype, shape, g):
    """Pages of keys and values with N(0, 1) entries, in 8 or 4 bits with their scales where held says so."""
    pool = {"k_scale": None, "v_scale": None}
    for n in "kv":
        x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)
        if held == "e4m3":
            x, pool[n + "_scale"] = _e4m3(x.float())
        elif held == "e2m1":
            v, pool[n + "_scale"] = _mx(x.float())
            x = _mx_codes(v).view(torch.float4_e2m1fn_x2)
        pool[n + "_pages"] = x
    return pool


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    def channels(n):
        # a few large channels, as activations and keys have them
        return 1.0 + 15.0 * (torch.rand(n, generator=g, device=DEV) < 0.03)

    if case["kind"] == "pack":
        return {"case": case, "x": (randn(case["m"], case["k"]) * channels(case["k"])).to(dtype)}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        v, scale = _mx(torch.randn((n, k), generator=g, device=DEV) * k ** -0.5)
        return {"case": case, "x": (randn(m, k) * channels(k)).to(dtype), "w": _mx_codes(v).view(torch.float4_e2m1fn_x2),
                "w_scale": scale, "bias": randn(n) if case["bias"] else None}
    chunks, lens = _lengths(case)
    width = -(-max(lens) // case["page"])
    need = [-(-n // case["page"]) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    rows, at = [], 0
    for n in need:
        rows.append(torch.cat([order[at:at + n], order.new_zeros(width - n)]))
        at += n
    starts = [sum(chunks[:i]) for i in range(len(chunks) + 1)]
    hkv, d = case["hkv"], case["d"]
    state = {"case": case, "table": torch.stack(rows), "starts": torch.tensor(starts, dtype=torch.int32, device=DEV),
             "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "max_q": max(chunks), "max_len": max(lens),
             **_pool("e2m1" if case["kind"] == "attend" else case["held"], dtype, (pages, hkv, case["page"], d), g),
             "q": randn(starts[-1], hkv * case["g"], d)}
    if case["kind"] == "append":
        sections = [int(x) for x in case["sections"].split(",")]
        state["freqs"] = torch.tensor([10000.0 ** (-i / s) for s in sections for i in range(s)], dtype=torch.float64, device=DEV)
        state["axes"] = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], dtype=torch.int32, device=DEV)
        state["pos"] = None
        if case["pos"]:  # far into a stream, as after hours of video, on each axis
            state["pos"] = torch.randint(0, 1 << 20, (starts[-1], len(sections)), generator=g, device=DEV, dtype=torch.int32)
        state["k"] = (randn(starts[-1], hkv, d) * channels(d)).to(dtype)
        state["v"] = randn(starts[-1], hkv, d)
    return state


# ------------------------------------------------------------------------------------------------- one pass


def _places(s):
    """Of each new token: its sequence's position, its page and slot."""
    t = torch.arange(s["k"].shape[0], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["starts"][1:], t, right=True)
    at = s["lens"][b] - s["starts"][b + 1] + t
    return at, s["table"][b, (at // s["case"]["page"]).long()].long(), (at % s["case"]["page"]).long()


def _plain_turn(s, x, at):
    """x's pairs turned, in 64 bits: codes next to a border between two are at stake."""
    p, adjacent = s["freqs"].numel(), s["case"]["pairs"] == "adjacent"
    pos = at[:, None] if s["pos"] is None else s["pos"][:, s["axes"].long()]
    angle = pos.double() * s["freqs"]
    c, sn, x = angle.cos()[:, None], angle.sin()[:, None], x.double()
    a, b = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if adjacent else (x[..., :p], x[..., p:2 * p])
    u, w = a * c - b * sn, b * c + a * sn
    turned = torch.stack([u, w], -1).flatten(-2) if adjacent else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., 2 * p:]], -1)


def _plain_write(s, x, name, page, slot):
    pages, scale = s[name + "_pages"], s[name + "_scale"]
    if scale is None:
        pages[page, :, slot] = x.to(pages.dtype)
        return
    if s["case"]["held"] == "e4m3":
        codes, exponents = _e4m3(x)
        codes = codes.view(torch.uint8)
    else:
        v, exponents = _mx(x)
        codes = _mx_codes(v)
    pages.view(torch.uint8)[page, :, slot] = codes
    scale[page, :, slot] = exponents


def _plain_dense(s, name):
    """What the sequences hold, [b, max_len, heads, d] in 32 bits, zeros behind each one's end."""
    pages, scale, ps = s[name + "_pages"], s[name + "_scale"], s["case"]["page"]
    at = torch.arange(s["max_len"], device=DEV)
    page, slot = s["table"][:, at // ps].long(), at % ps
    codes, scale = pages.view(torch.uint8)[page, :, slot], scale[page, :, slot]
    if pages.dtype == torch.float8_e4m3fn:
        x = codes.view(torch.float8_e4m3fn).float() * _power(scale.int() - 127)[..., None]
    else:
        x = _mx_values(codes, scale)
    return torch.where((at < s["lens"][:, None])[..., None, None], x, 0.0)


def _plain_append(s):
    at, page, slot = _places(s)
    _plain_write(s, _plain_turn(s, s["k"], at), "k", page, slot)
    _plain_write(s, s["v"].double(), "v", page, slot)
    q = _plain_turn(s, s["q"], at).to(s["q"].dtype)
    if s["k_scale"] is None:
        return q, s["k_pages"], s["v_pages"]
    return (q, *(_plain_dense(s, n).to(q.dtype) for n in "kv"))


def _plain_attention(s):
    case, q = s["case"], s["q"]
    b, hkv, g, d, mq = case["b"], case["hkv"], case["g"], case["d"], s["max_q"]
    k, v = (_plain_dense(s, n) for n in "kv")
    chunk = s["starts"][1:] - s["starts"][:-1]
    i = torch.arange(mq, device=DEV)
    rows = (s["starts"][:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q.float()[rows].view(b, mq, hkv, g, d).transpose(1, 2).reshape(b * hkv, mq * g, d)
    kt = k.permute(0, 2, 3, 1).reshape(b * hkv, d, -1).contiguous()
    scores = torch.bmm(qp * d ** -0.5, kt).view(b, hkv, mq, g, -1)
    last = (s["lens"] - chunk)[:, None] + i + 1 if case["causal"] else s["lens"][:, None].expand(b, mq)
    seen = torch.arange(s["max_len"], device=DEV) < last[:, None, :, None, None]
    scores = torch.where(seen, scores, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(b * hkv, mq * g, -1), v.transpose(1, 2).reshape(b * hkv, -1, d).contiguous())
    o = o.view(b, hkv, mq, g, d).transpose(1, 2).reshape(b, mq, hkv * g, d)
    return o[i < chunk[:, None]].to(q.dtype)


def _plain_linear(s):
    v, scale = _mx(s["x"].float())
    x = (v * torch.where(scale == 255, float("nan"), _power(scale.int().clamp(max=254) - 127))[..., None]).flatten(-2)
    y = torch.mm(x, _mx_values(s["w"].view(torch.uint8), s["w_scale"]).T.contiguous())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    return y.to(s["x"].dtype)


def run(s):
    case = s["case"]
    if own:
        hip = _hip()
        if case["kind"] == "pack":
            return hip.mx_unpack(*hip.mx_pack(s["x"]), dtype=s["x"].dtype)
        if case["kind"] == "linear":
            return hip.mx_linear(s["x"], s["w"], s["w_scale"], s["bias"], gelu=case["gelu"])
        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if case["kind"] == "attend":
            return hip.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["lens"],
                                       causal=case["causal"], max_q=s["max_q"], max_len=s["max_len"], **scales)
        q = hip.kv_append(s["q"], s["k"], s["v"], s["freqs"], s["axes"], s["k_pages"], s["v_pages"], s["table"], s["starts"],
                          s["lens"], pos=s["pos"], pairs=case["pairs"], **scales)
        if s["k_scale"] is None:
            return q, s["k_pages"], s["v_pages"]
        return (q, *hip.kv_read(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["max_len"], dtype=q.dtype, **scales))
    if case["kind"] == "pack":
        v, scale = _mx(s["x"].float())
        return _mx_values(_mx_codes(v), scale).to(s["x"].dtype)
    if case["kind"] == "linear":
        return _plain_linear(s)
    return _plain_append(s) if case["kind"] == "append" else _plain_attention(s)


# ------------------------------------------------------------------------------------------------- 64 bits


def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest(x, top, mantissa, low):
    """Values of blocks (the last dimension) of x to the nearest (ties to even) multiples of 2^(e - mantissa) times their
    power of two, the least that holds the block's largest below `top` of it; e is the binary exponent of the scaled value,
    `low` at least."""
    largest = x.abs().amax(-1, keepdim=True)
    e = torch.frexp(largest / top)[1].long()  # the quotient is below 2^e; one step less where it is 2^(e-1) itself
    e = torch.where(largest <= top * _two_to(e - 1), e - 1, e)
    s = torch.where(largest > 0, _two_to(e), 1.0)
    y = x / s
    step = _two_to((torch.frexp(y)[1].long() - 1).clamp(min=low) - mantissa)
    return torch.round(y / step) * step * s


def _four_bits(x):
    return _nearest(x.double().view(*x.shape[:-1], -1, BLOCK), E2M1_MAX, 1, 0).view(x.shape)


def _held(pages, scale, of):
    """64-bit values of some pages."""
    if scale is None:
        return pages[of].double()
    if pages.dtype == torch.float8_e4m3fn:
        return pages[of].double() * _two_to(scale[of].long() - 127)[..., None]
    c = pages.view(torch.uint8)[of].long()
    c = torch.stack([c % 16, c // 16], -1).flatten(-2)
    m, e = c % 2, c // 2 % 4  # (1 + m / 2) 2^(e - 1), or m / 2 where e is 0
    x = torch.where(e > 0, (1 + 0.5 * m) * _two_to(e - 1), 0.5 * m.double()) * (1 - 2 * (c // 8))
    return x * _two_to(scale[of].long() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pack":
        return _four_bits(s["x"])
    if case["kind"] == "linear":
        y = _four_bits(s["x"]) @ _held(s["w"], s["w_scale"], slice(None)).T.contiguous()
        if s["bias"] is not None:
            y += s["bias"].double()
        return y * 0.5 * torch.erfc(-y / math.sqrt(2.0)) if case["gelu"] else y
    ps, starts, lens = case["page"], s["starts"].tolist(), s["lens"].tolist()
    hkv, d = case["hkv"], case["d"]
    if case["kind"] == "append":
        at = [n - (starts[i + 1] - starts[i]) + j for i, n in enumerate(lens) for j in range(starts[i + 1] - starts[i])]
        at = torch.tensor(at, device=DEV)
        turned = {}
        for name in "qk":
            x = s[name].double()
            out, p = x.clone(), s["freqs"].numel()
            for i in range(p):
                where = at if s["pos"] is None else s["pos"][:, int(s["axes"][i])]
                angle = (where.double() * s["freqs"][i])[:, None]
                lo, hi = (2 * i, 2 * i + 1) if case["pairs"] == "adjacent" else (i, i + p)
                out[..., lo] = x[..., lo] * torch.cos(angle) - x[..., hi] * torch.sin(angle)
                out[..., hi] = x[..., hi] * torch.cos(angle) + x[..., lo] * torch.sin(angle)
            turned[name] = out
        outs = [turned["q"]]
        for name, new in (("k", turned["k"]), ("v", s["v"].double())):
            pages, scale = s[name + "_pages"], s[name + "_scale"]
            if case["held"] == "e4m3":
                new = _nearest(new, E4M3_MAX, 3, -6)
            elif case["held"] == "e2m1":
                new = _four_bits(new)
            out = pages.double() if scale is None else torch.zeros(case["b"], s["max_len"], hkv, d, device=DEV, dtype=torch.float64)
            for i, length in enumerate(lens):
                held = s["table"][i, : -(-length // ps)].long()
                rows = _held(pages, scale, held).transpose(1, 2).reshape(-1, hkv, d)
                rows[length - (starts[i + 1] - starts[i]):length] = new[starts[i]:starts[i + 1]]
                if scale is None:
                    out[held] = rows.view(-1, ps, hkv, d).transpose(1, 2)
                else:
                    out[i, :length] = rows[:length]
            outs.append(out)
        return tuple(outs)
    outs = []
    for i, length in enumerate(lens):
        held = s["table"][i, : -(-length // ps)].long()
        k, v = (_held(s[n + "_pages"], s[n + "_scale"], held).transpose(0, 1).reshape(hkv, -1, d)[:, :length] for n in "kv")
        q = s["q"][starts[i]:starts[i + 1]].double()
        n = q.shape[0]
        out = torch.empty_like(q)
        for h in range(q.shape[1]):
            w = (q[:, h] @ k[h // case["g"]].T.contiguous()) * d ** -0.5
            if case["causal"]:
                w = w.masked_fill(torch.ones(n, length, device=DEV, dtype=torch.bool).triu(length - n + 1), float("-inf"))
            out[:, h] = torch.softmax(w, -1) @ v[h // case["g"]]
        outs.append(out)
    return torch.cat(outs)


# ------------------------------------------------------------------------------------------------- work


def work(case):
    elem = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "pack":
        n = case["m"] * case["k"]
        return {"bytes": 2 * n * elem + 2 * n * 17 // 32, "flops": 2 * n}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + m * n + (n if case["bias"] else 0)) * elem + n * k * 17 // 32, "flops": 2 * m * n * k}
    chunks, lens = _lengths(case)
    d, hkv, heads = case["d"], case["hkv"], case["hkv"] * case["g"]
    held = "e2m1" if case["kind"] == "attend" else case["held"]
    row = d * 17 // 32 if held == "e2m1" else d + 1 if held == "e4m3" else d * elem  # a held row of one head, its scales included
    tables = sum(4 * -(-n // case["page"]) for n in lens) + 4 * (2 * case["b"] + 1)
    if case["kind"] == "append":
        new = sum(chunks)
        pairs, axes = sum(int(x) for x in case["sections"].split(",")), case["sections"].count(",") + 1
        n = new * (2 * heads + 2 * hkv) * d * elem + 2 * new * hkv * row + (4 * new * axes if case["pos"] else 0) + 12 * pairs
        if held != "own":  # what the sequences hold is read back
            n += 2 * hkv * (sum(lens) * row + case["b"] * max(lens) * d * elem)
        return {"bytes": n + tables, "flops": 6 * new * (heads + hkv) * pairs}
    seen = sum(c * n - (c * (c - 1) // 2 if case["causal"] else 0) for c, n in zip(chunks, lens))
    return {"bytes": 2 * sum(chunks) * heads * d * elem + 2 * sum(lens) * hkv * row + tables, "flops": 4 * d * heads * seen}
