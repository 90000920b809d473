"""The paged memory's operators in 64 bits on the CPU, from their definitions, and the bounds that the tests hold
kernels to. Nothing here uses the library."""
import math

import torch

E4M3_MAX = 448.0
F32_U = 2.0 ** -24  # half a step of f32, relative


def rope(x, pos, freqs, axes, pairs="adjacent", inverse=False):
    """x [..., L, H, D] f64, pos [..., L, A]."""
    x, out = x.double(), x.double().clone()
    p = len(freqs)
    for i in range(p):
        a = (pos[..., int(axes[i])].double() * float(freqs[i]) * (-1 if inverse else 1))[..., None]
        lo, hi = (2 * i, 2 * i + 1) if pairs == "adjacent" else (i, i + p)
        out[..., lo] = x[..., lo] * a.cos() - x[..., hi] * a.sin()
        out[..., hi] = x[..., hi] * a.cos() + x[..., lo] * a.sin()
    return out


def rope_bound(x, want, pairs_n, pairs, dtype):
    """Sine and cosine: the fraction of a turn rounds once (2^-26 turns, 9.4e-8), its product with 2 pi twice (9.4e-8
    on an eighth of a turn), the Taylor sums by 1.5 half steps (9e-8): below 2.8e-7 each. The turn's two f32 roundings
    add 2^-23 of |x0| + |x1|. Then the output's own rounding."""
    x = x.double().abs()
    s = torch.zeros_like(x)
    if pairs == "adjacent":
        t = x[..., 0:2 * pairs_n:2] + x[..., 1:2 * pairs_n:2]
        s[..., 0:2 * pairs_n:2], s[..., 1:2 * pairs_n:2] = t, t
    else:
        t = x[..., :pairs_n] + x[..., pairs_n:2 * pairs_n]
        s[..., :pairs_n], s[..., pairs_n:2 * pairs_n] = t, t
    return 4.0e-7 * s + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def quantise(x):
    """(values that the codes stand for, biased scale exponents) of rows of x."""
    x = x.double()
    fin = torch.isfinite(x)
    top = torch.where(fin, x.abs(), torch.zeros_like(x)).amax(-1)
    s = torch.zeros(top.shape, dtype=torch.int64)
    flat, out = top.reshape(-1).tolist(), s.reshape(-1)
    for i, t in enumerate(flat):
        if t > 0:
            e = math.frexp(t / E4M3_MAX)[1]  # t / 448 < 2^e; two candidates, the smaller that holds it
            e = e - 1 if t <= E4M3_MAX * 2.0 ** (e - 1) else e
            out[i] = max(-126, min(126, e))
    two = torch.pow(torch.tensor(2.0, dtype=torch.float64), s.double())[..., None]
    y = torch.where(fin, x, torch.zeros_like(x)) / two
    e = (torch.frexp(y)[1].long() - 1).clamp(min=-6)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 3).double())
    val = torch.round(y / step) * step * two  # torch.round: ties to even
    return torch.where(fin, val, torch.full_like(val, float("nan"))), (s + 127).to(torch.uint8)


def positions(starts, lens, b):
    """Position of each of sequence b's new tokens."""
    n = starts[b + 1] - starts[b]
    return [lens[b] - n + i for i in range(n)]


def gather(pages, table, b, length, page):
    """Sequence b's rows [length, heads, d]; rows of pages that are not there are None-d by the mask."""
    rows, there = [], []
    for j in range(length):
        e = int(table[b][j // page])
        ok = 0 <= e < pages.shape[0]
        there.append(ok)
        rows.append(pages[e, :, j % page] if ok else torch.zeros_like(pages[0, :, 0]))
    if not rows:
        return pages.new_zeros(0, pages.shape[1], pages.shape[3]), torch.zeros(0, dtype=torch.bool)
    return torch.stack(rows), torch.tensor(there)


def attention(q, k_pages, v_pages, table, starts, lens, scale, causal, p_unit):
    """(out, bound) in f64 for rows of every sequence; rows of none are NaN in both. p_unit: the relative rounding that
    the kernel's P has before it meets v (0 in f32). Non-finite v counts where its key is seen."""
    q = q.double()
    t, hq, d = q.shape
    hkv, page = k_pages.shape[1], k_pages.shape[2]
    g = hq // hkv
    out = torch.full_like(q, float("nan"))
    bound = torch.full_like(q, float("nan"))
    for b in range(len(lens)):
        length = max(0, min(int(lens[b]), table.shape[1] * page))
        k, there = gather(k_pages.double(), table, b, length, page)
        v, _ = gather(v_pages.double(), table, b, length, page)
        n = starts[b + 1] - starts[b]
        for i in range(n):
            row = starts[b] + i
            last = max(0, min(length, length - n + i + 1)) if causal else length
            see = there[:last].nonzero().flatten()
            for h in range(hq):
                kk, vv = k[see][:, h // g], v[see][:, h // g]
                if len(see) == 0:
                    out[row, h], bound[row, h] = 0.0, 0.0
                    continue
                s = (kk @ q[row, h]) * scale
                w = torch.softmax(s, 0)
                out[row, h] = (w[:, None] * vv).sum(0)
                # each score is off by at most (d + 2) roundings of its absolute products, each weight by twice that
                # (numerator and denominator), P's rounding twice likewise, and the sums by one rounding a key
                mass = float((kk.abs() @ q[row, h].abs()).max()) * scale if torch.isfinite(kk).all() else 0.0
                rel = 2 * (d + 2) * F32_U * mass + 2 * p_unit + (len(see) + 16) * F32_U
                bound[row, h] = rel * (w[:, None] * vv.abs()).sum(0)
    return out, bound


def with_rounding(bound, want, dtype):
    """A bound with the rounding of the output to its type."""
    f = torch.finfo(dtype)
    return bound + f.eps / 2 * (want.abs() + bound) + f.smallest_normal * f.eps / 2
