"""Performance cases of the paged key/value memory: rotary positions over several axes, the cache's writing and
reading back, and the attention of new tokens over it.

Three kinds of work:

    rope     rope_axes: queries or keys turned by their (time, row, column) positions
    cache    kv_write of a chunk of new tokens into its pages, then kv_read of what the sequences hold
    attend   paged_attention of each sequence's new tokens over its pages

listed() holds sizes that a video's memory bank and a server's decoding have; draw() gives others of the same ranges.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
E4M3_MAX = 448.0


def _hip():
    if "sam_hip" not in sys.modules:  # a program imports it once
        sys.path.insert(0, os.path.abspath("sam-rs_amd"))
        import sam_hip  # noqa: F401
    return sys.modules["sam_hip"]


def listed():
    return [
        # One new token's keys at (time, row, column): what a decoding step turns. The smallest call, latency.
        {"name": "rope_token_bf16", "kind": "rope", "dtype": "bf16", "n": 1, "h": 8, "d": 64, "sections": "8,12,12",
         "pairs": "halves"},
        # The keys of one 64 x 64 frame of a video's memory (SAM 2.1: one head of 256), with a time axis.
        {"name": "rope_frame_f16", "kind": "rope", "dtype": "f16", "n": 4096, "h": 1, "d": 256, "sections": "32,48,48",
         "pairs": "adjacent"},
        # A clip of 8 frames of 72 x 72 patches, 16 heads of 64 (SAM 3's ViT): the largest.
        {"name": "rope_clip_f16", "kind": "rope", "dtype": "f16", "n": 41472, "h": 16, "d": 64, "sections": "8,12,12",
         "pairs": "adjacent"},
        # A decoding step of 32 sequences into 8 bits, each with a short history that is read back.
        {"name": "cache_steps_fp8_bf16", "kind": "cache", "dtype": "bf16", "fp8": True, "b": 32, "chunk": 1, "len": 40,
         "ragged": 0.8, "hkv": 8, "d": 128, "page": 16},
        # A frame of 4096 tokens enters a video's memory of 7 frames and 64 pointer tokens, which is read back.
        {"name": "cache_frame_fp8_f16", "kind": "cache", "dtype": "f16", "fp8": True, "b": 1, "chunk": 4096,
         "len": 28736, "ragged": 0.0, "hkv": 1, "d": 256, "page": 64},
        # Four objects' prompts of odd lengths into 16-bit pages that are no power of two, and back.
        {"name": "cache_prompts_f16", "kind": "cache", "dtype": "f16", "fp8": False, "b": 4, "chunk": 1000, "len": 3001,
         "ragged": 0.7, "hkv": 5, "d": 80, "page": 24},
        # One token over a short history, 8 heads of 64: latency.
        {"name": "attend_token_f16", "kind": "attend", "dtype": "f16", "fp8": False, "b": 1, "chunk": 1, "len": 577,
         "ragged": 0.0, "hkv": 8, "g": 1, "d": 64, "page": 16, "causal": True},
        # A server's decoding step: 32 sequences of up to 8192 tokens in 8 bits, 32 query and 8 key heads of 128.
        {"name": "attend_steps_fp8_bf16", "kind": "attend", "dtype": "bf16", "fp8": True, "b": 32, "chunk": 1,
         "len": 8192, "ragged": 0.9, "hkv": 8, "g": 4, "d": 128, "page": 16, "causal": True},
        # One token over a long history, 16 query and 2 key heads of 128.
        {"name": "attend_long_f16", "kind": "attend", "dtype": "f16", "fp8": False, "b": 1, "chunk": 1, "len": 131072,
         "ragged": 0.0, "hkv": 2, "g": 8, "d": 128, "page": 64, "causal": True},
        # SAM 2.1's memory attention, cross: a frame's 4096 queries over 7 frames and 64 pointer tokens, in 8 bits.
        {"name": "attend_memory_fp8_f16", "kind": "attend", "dtype": "f16", "fp8": True, "b": 1, "chunk": 4096,
         "len": 28736, "ragged": 0.0, "hkv": 1, "g": 1, "d": 256, "page": 64, "causal": False},
        # Chunks of 5 prompts of different lengths over their histories, 16 query and 4 key heads of 128.
        {"name": "attend_chunks_bf16", "kind": "attend", "dtype": "bf16", "fp8": False, "b": 5, "chunk": 1024,
         "len": 8192, "ragged": 0.8, "hkv": 4, "g": 4, "d": 128, "page": 16, "causal": True},
        # Six tracked objects, 32 x 32 queries each over memories of different ages, pages that end inside tiles.
        {"name": "attend_objects_f16", "kind": "attend", "dtype": "f16", "fp8": False, "b": 6, "chunk": 1024,
         "len": 7000, "ragged": 0.7, "hkv": 8, "g": 1, "d": 64, "page": 24, "causal": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    kind = rng.choice(["rope", "cache", "cache", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["f16", "f16", "f16", "bf16", "bf16", "bf16", "f32"])
    if kind == "rope":
        d = 8 * rng.randint(4, 32)
        a = rng.choice([2, 3])
        rows = rng.randint(1, d // 4 - 1)
        time = rng.randint(1, d // 2 - rows - 1) if a == 3 else 0
        cols = d // 2 - rows - time if rng.random() < 0.7 else rng.randint(1, d // 2 - rows - time)
        return {"kind": kind, "dtype": dtype, "n": _log(rng, 1, 65536), "h": _log(rng, 1, 16), "d": d,
                "sections": ",".join(str(x) for x in ([time] if time else []) + [rows, cols]),
                "pairs": rng.choice(["adjacent", "halves"])}
    b = _log(rng, 1, 64)
    length = _log(rng, 1, 65536)
    case = {"kind": kind, "dtype": dtype, "fp8": rng.random() < 0.5, "b": b,
            "chunk": min(length, rng.choice([1, 1, _log(rng, 1, 4096)])), "len": length,
            "ragged": rng.choice([0.0, 0.5, 0.9]), "hkv": _log(rng, 1, 16), "d": rng.choice([64, 72, 80, 96, 128, 256]),
            "page": rng.choice([8, 16, 24, 32, 64, 100, 128, 256])}
    if kind == "attend":
        case["g"] = rng.choice([1, 1, 2, 3, 4, 6, 8])
        case["causal"] = rng.random() < 0.6
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / (1e14 if case["dtype"] == "f32" else 1e15))


def _room(case):
    """Bytes that the plain form holds at most: the keys and values and the scores of a padded batch in 32 bits."""
    if case["kind"] == "rope":
        return 0
    n = 4 * 4 * case["b"] * case["hkv"] * case["len"] * case["d"]
    if case["kind"] == "attend":
        n += 3 * 4 * case["b"] * case["hkv"] * case["g"] * case["chunk"] * case["len"]
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


def _power(s):
    """2^s in 32 bits, exactly, for whole s from -126 to 127."""
    return ((s + 127).to(torch.int32) << 23).view(torch.float32)


def _quantised(x):
    """e4m3 codes of rows and the biased exponents of their scales, the powers of two that bring a row's largest
    value to 448 at most and as near to it as they can."""
    x = x.float()
    m, e = torch.frexp(torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1))
    s = torch.where(m > 0, e - 9 + (m > E4M3_MAX / 512).int(), 0).clamp(-126, 126)
    return (x * _power(-s)[..., None]).to(torch.float8_e4m3fn), (s + 127).to(torch.uint8)


def _pool(case, pages, g):
    """Pages of keys and values with N(0, 1) entries, in 8 bits with their scales where the case says so."""
    shape = (pages, case["hkv"], case["page"], case["d"])
    k, v = (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(DTYPES[case["dtype"]]) for _ in range(2))
    if not case["fp8"]:
        return {"k_pages": k, "v_pages": v, "k_scale": None, "v_scale": None}
    (k, ks), (v, vs) = _quantised(k), _quantised(v)
    return {"k_pages": k, "v_pages": v, "k_scale": ks, "v_scale": vs}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    if case["kind"] == "rope":
        sections = [int(x) for x in case["sections"].split(",")]
        freqs = [10000.0 ** (-i / s) for s in sections for i in range(s)]
        axes = [a for a, s in enumerate(sections) for i in range(s)]
        return {"case": case, "x": randn(1, case["n"], case["h"], case["d"]),
                # positions far into a stream, as after hours of video, on each axis
                "pos": torch.randint(0, 1 << 20, (1, case["n"], len(sections)), generator=g, device=DEV, dtype=torch.int32),
                "freqs": torch.tensor(freqs, dtype=torch.float64, device=DEV),
                "axes": torch.tensor(axes, dtype=torch.int32, device=DEV)}
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
    state = {"case": case, "table": torch.stack(rows), "starts": torch.tensor(starts, dtype=torch.int32, device=DEV),
             "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "max_q": max(chunks), "max_len": max(lens),
             **_pool(case, pages, g)}
    if case["kind"] == "cache":
        # activations with a few large channels, as keys have them
        big = 1.0 + 15.0 * (torch.rand(case["d"], generator=g, device=DEV) < 0.03)
        state["k"] = (randn(starts[-1], case["hkv"], case["d"]) * big).to(dtype)
        state["v"] = randn(starts[-1], case["hkv"], case["d"])
    else:
        state["q"] = randn(starts[-1], case["hkv"] * case["g"], case["d"])
    return state


# ------------------------------------------------------------------------------------------------- one pass


def _plain_rope(s):
    x, p, adjacent = s["x"].float(), s["freqs"].numel(), s["case"]["pairs"] == "adjacent"
    angle = s["pos"][..., s["axes"].long()].double() * s["freqs"]
    c, sn = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    a, b = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if adjacent else (x[..., :p], x[..., p:2 * p])
    u, w = a * c - b * sn, b * c + a * sn
    turned = torch.stack([u, w], -1).flatten(-2) if adjacent else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., 2 * p:]], -1).to(s["x"].dtype)


def _plain_write(s, x, pages, scale):
    ps = s["case"]["page"]
    t = torch.arange(x.shape[0], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["starts"][1:], t, right=True)
    at = (s["lens"][b] - s["starts"][b + 1] + t).long()
    page, slot = s["table"][b, at // ps].long(), at % ps
    if scale is None:
        pages[page, :, slot] = x
        return
    codes, exponents = _quantised(x)
    pages.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
    scale[page, :, slot] = exponents


def _plain_dense(s, pages, scale):
    """What the sequences hold, [b, max_len, heads, d] in 32 bits, zeros behind each one's end."""
    ps = s["case"]["page"]
    at = torch.arange(s["max_len"], device=DEV)
    page, slot = s["table"][:, at // ps].long(), at % ps
    if scale is None:
        x = pages[page, :, slot].float()
    else:
        codes = pages.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn)
        x = codes.float() * _power(scale[page, :, slot].int() - 127)[..., None]
    return torch.where((at < s["lens"][:, None])[..., None, None], x, 0.0)


def _plain_attention(s):
    case, q = s["case"], s["q"]
    b, hkv, g, d, mq = case["b"], case["hkv"], case["g"], case["d"], s["max_q"]
    k, v = (_plain_dense(s, s[n + "_pages"], s[n + "_scale"]) for n in "kv")
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


def run(s):
    case = s["case"]
    if own:
        hip = _hip()
        if case["kind"] == "rope":
            return hip.rope_axes(s["x"], s["pos"], s["freqs"], s["axes"], pairs=case["pairs"])
        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if case["kind"] == "cache":
            hip.kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["lens"], **scales)
            return hip.kv_read(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["max_len"],
                               dtype=s["k"].dtype, **scales)
        return hip.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["lens"],
                                   causal=case["causal"], max_q=s["max_q"], max_len=s["max_len"], **scales)
    if case["kind"] == "rope":
        return _plain_rope(s)
    if case["kind"] == "cache":
        _plain_write(s, s["k"], s["k_pages"], s["k_scale"])
        _plain_write(s, s["v"], s["v_pages"], s["v_scale"])
        return tuple(_plain_dense(s, s[n + "_pages"], s[n + "_scale"]).to(s["k"].dtype) for n in "kv")
    return _plain_attention(s)


# ------------------------------------------------------------------------------------------------- 64 bits


def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _value(pages, scale):
    x = pages.double()
    return x if scale is None else x * _two_to(scale.long() - 127)[..., None]


def _e4m3_values(x):
    """The values that rows of x stand for in 8 bits: nearest (ties to even) multiples of 2^(e-3) times the row's scale,
    e the binary exponent of the scaled value and -6 at least."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.frexp(top / E4M3_MAX)[1].long()  # the quotient is below 2^e; one step less where it is 2^(e-1) itself
    e = torch.where(top <= E4M3_MAX * _two_to(e - 1), e - 1, e)
    s = torch.where(top > 0, _two_to(e), 1.0)
    y = x / s
    step = _two_to((torch.frexp(y)[1].long() - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step * s


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        x = s["x"].double()
        out, adjacent, p = x.clone(), case["pairs"] == "adjacent", s["freqs"].numel()
        for i in range(p):
            angle = (s["pos"][:, :, int(s["axes"][i])].double() * s["freqs"][i])[..., None]
            lo, hi = (2 * i, 2 * i + 1) if adjacent else (i, i + p)
            out[..., lo] = x[..., lo] * torch.cos(angle) - x[..., hi] * torch.sin(angle)
            out[..., hi] = x[..., hi] * torch.cos(angle) + x[..., lo] * torch.sin(angle)
        return out
    ps, starts, lens = case["page"], s["starts"].tolist(), s["lens"].tolist()
    if case["kind"] == "cache":
        both = []
        for n in "kv":
            out = torch.zeros(case["b"], s["max_len"], case["hkv"], case["d"], device=DEV, dtype=torch.float64)
            new = _e4m3_values(s[n]) if case["fp8"] else s[n].double()
            for i, length in enumerate(lens):
                held = s["table"][i, : -(-length // ps)].long()
                x = _value(s[n + "_pages"][held], None if s[n + "_scale"] is None else s[n + "_scale"][held])
                x = x.transpose(1, 2).reshape(-1, case["hkv"], case["d"])[:length]
                x[length - (starts[i + 1] - starts[i]):] = new[starts[i]:starts[i + 1]]
                out[i, :length] = x
            both.append(out)
        return tuple(both)
    outs = []
    for i, length in enumerate(lens):
        held = s["table"][i, : -(-length // ps)].long()
        k, v = (_value(s[n + "_pages"][held], None if s[n + "_scale"] is None else s[n + "_scale"][held])
                .transpose(0, 1).reshape(case["hkv"], -1, case["d"])[:, :length] for n in "kv")
        q = s["q"][starts[i]:starts[i + 1]].double()
        n = q.shape[0]
        out = torch.empty_like(q)
        for h in range(q.shape[1]):
            w = (q[:, h] @ k[h // case["g"]].T.contiguous()) * case["d"] ** -0.5
            if case["causal"]:
                w = w.masked_fill(torch.ones(n, length, device=DEV, dtype=torch.bool).triu(length - n + 1), float("-inf"))
            out[:, h] = torch.softmax(w, -1) @ v[h // case["g"]]
        outs.append(out)
    return torch.cat(outs)


# ------------------------------------------------------------------------------------------------- work


def work(case):
    elem = 4 if case["dtype"] == "f32" else 2
    d = case["d"]
    if case["kind"] == "rope":
        pairs = sum(int(x) for x in case["sections"].split(","))
        n, axes = case["n"], case["sections"].count(",") + 1
        return {"bytes": 2 * n * case["h"] * d * elem + 4 * n * axes + 12 * pairs, "flops": 6 * n * case["h"] * pairs}
    chunks, lens = _lengths(case)
    row = d + 1 if case["fp8"] else d * elem  # a held row of one head, its scale included
    tables = sum(4 * -(-n // case["page"]) for n in lens) + 4 * (2 * case["b"] + 1)
    if case["kind"] == "cache":
        new, held = sum(chunks) * case["hkv"], sum(lens) * case["hkv"]
        padded = case["b"] * max(lens) * case["hkv"]
        return {"bytes": 2 * (new * (d * elem + row) + held * row + padded * d * elem) + tables, "flops": 2 * new * d}
    seen = sum(c * n - (c * (c - 1) // 2 if case["causal"] else 0) for c, n in zip(chunks, lens))
    heads = case["hkv"] * case["g"]
    return {"bytes": 2 * sum(chunks) * heads * d * elem + 2 * sum(lens) * case["hkv"] * row + tables,
            "flops": 4 * d * heads * seen}
