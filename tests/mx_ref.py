"""4-bit numbers in scaled blocks and their products in 64 bits on the CPU, from their definitions, and the bounds that the
tests hold kernels to. Nothing here uses the library."""
import math

import torch

BLOCK = 32
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
F64 = torch.float64


def two_to(s):
    return torch.pow(torch.tensor(2.0, dtype=F64), s.double())


def quantise(x):
    """(values, codes one a byte, scale bytes) of rows of x in blocks of 32."""
    y = x.double().unflatten(-1, (-1, BLOCK))
    fine = torch.isfinite(y).all(-1)
    y = torch.where(fine[..., None], y, torch.zeros_like(y))
    top = y.abs().amax(-1)
    s = torch.zeros(top.shape, dtype=torch.int64)
    flat = s.view(-1)
    for i, t in enumerate(top.reshape(-1).tolist()):
        if t > 0:
            e = math.frexp(t / 6.0)[1]  # t / 6 < 2^e; two candidates, the smaller that holds it
            flat[i] = max(-126, min(126, e - 1 if t <= 6.0 * 2.0 ** (e - 1) else e))
    z = y / two_to(s)[..., None]
    grid = torch.tensor(GRID, dtype=F64)
    # the nearest value; of two as near, the one with an even code
    off = (z.abs()[..., None] - grid).abs()
    near = off.amin(-1, keepdim=True)
    code = torch.arange(8)
    even = torch.where(off == near, code % 2, 2)
    pick = even.argmin(-1)
    value = grid[pick] * torch.where(torch.signbit(z), -1.0, 1.0) * two_to(s)[..., None]
    value = torch.where(fine[..., None], value, torch.full_like(value, float("nan")))
    codes = torch.where(fine[..., None], pick + 8 * torch.signbit(z).long(), torch.zeros_like(pick))
    return value.flatten(-2), codes.flatten(-2).to(torch.uint8), torch.where(fine, s + 127, 255).to(torch.uint8)


def packed(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values(codes, scale):
    """What packed codes (any dtype of one byte) and scale bytes stand for, in 64 bits."""
    c = codes.cpu().view(torch.uint8)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).long()
    grid = torch.tensor(GRID + [-g for g in GRID], dtype=F64)
    s = scale.cpu().long()
    two = torch.where(s == 255, torch.full(s.shape, float("nan"), dtype=F64), two_to(s - 127))
    return (grid[c].unflatten(-1, (-1, BLOCK)) * two[..., None]).flatten(-2)


def gelu(x):
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))


def product(a, b, bias, act, dtype):
    """(act(a b^T + bias), bound) for the kernel's f32 sums. Products are exact; k of them and the bias take k + 1 additions
    at most, in any order, each off by one step (2^-23) at most of a partial sum that the absolute products bound. The GELU
    passes an error on 1.13 times at most and adds that of erfc (a fit to 1.2e-7, its argument's roundings, 1e-6 of it in
    all) times x / 2. Then the rounding of the output to its type."""
    want, mass = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    bound = (a.shape[-1] + 1) * 2.0 ** -23 * mass
    if act:
        bound = 1.13 * bound + 0.5e-6 * (want.abs() + bound)
        want = gelu(want)
    f = torch.finfo(dtype)
    return want, bound + f.eps / 2 * (want.abs() + bound) + f.smallest_normal * f.eps / 2
