"""The GELU of 4-bit products alone: sums that are exact, so that the activation and the output's rounding are all that is off."""
import math

import pytest
import torch

import sam_hip

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def loaded():
    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"


def bound(x, want, dtype):
    """16 bits: the activation's relative error (1.1e-5, down to x = -12; below, its exponential is next to f32's smallest normal
    number, which it may fall to zero from) and half a step of the output. f32: erfc's fit of 1.2e-7, then the roundings of its
    argument z = |x| / sqrt 2 (two, so that z^2 is off by four half steps), of -z^2 + p (one), of the product with log2 e (two), of
    exp2 (two, an instruction of one step) and of 1 / (1 + z / 2), p and the products around them (thirty at most, p' below 2.2),
    each 2^-24 of a number that z^2 + 2 bounds where it is an exponent."""
    f = torch.finfo(dtype)
    if dtype == torch.float32:
        z2 = x * x / 2
        rel = 1.2e-7 + (7 * z2 + 44) * 2.0 ** -24
    else:
        rel = 1.1e-5
    off = rel * want.abs() + x.abs().clamp(max=14.0) * 2.0 ** -126
    return off + f.eps / 2 * (want.abs() + off) + f.smallest_normal * f.eps / 2


def check(got, x, dtype):
    x = x.double().cpu()
    want = 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))
    want = torch.where(x < -30, torch.zeros_like(x), want)  # x erfc(30) is below 2^-600
    off, most = (got.cpu().double() - want).abs(), bound(x, want, dtype)
    assert torch.isfinite(got).all()
    assert (off <= most).all(), (float(x.expand_as(off)[off > most][0]), float((off / most).max()))


def every(dtype):
    """Every finite value of a 16-bit type, or a sweep of f32's."""
    if dtype == torch.float32:
        g = torch.Generator().manual_seed(0)
        return torch.cat([torch.linspace(-13, 13, 60001), torch.randn(4000, generator=g) * 1e-3, torch.tensor([0.0, -0.0, 1e30, -1e30])])
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    return x[torch.isfinite(x)]


@pytest.mark.parametrize("m", [1, 20, 40, 300, 2000])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_of_every_value(m, dtype):
    """Rows of zeros, so that the sum is the bias: few rows, and tiles of all sizes."""
    dt = DT[dtype]
    x = every(dt).cuda()
    zeros = sam_hip.mx_pack(torch.zeros(m, 32, device="cuda"))
    got = sam_hip.mx_matmul(*zeros, *sam_hip.mx_pack(torch.zeros(len(x), 32, device="cuda")), x, gelu=True, dtype=dt)
    assert torch.equal(got, got[:1].expand_as(got))  # rows alike, bit for bit
    check(got[0], x, dt)


@pytest.mark.parametrize("m", [16, 64, 500])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_between_values_of_16_bits(m, dtype):
    """One product of two codes and two scales added to a bias: sums of up to 24 bits, exact in f32, from -11.5 to 11.5 + 36 / 32."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(1)
    a, b = torch.zeros(m, 32), torch.zeros(4096, 32)
    code = lambda n: torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[torch.randint(0, 7, (n,), generator=g)]
    a[:, 5], b[:, 5] = code(m) * torch.pow(2.0, -torch.randint(0, 3, (m,), generator=g).float()), code(4096) * torch.pow(2.0, -torch.randint(5, 12, (4096,), generator=g).float())
    bias = (torch.linspace(-11.5, 11.5, 4096) * 64).round().div(64).to(dt)  # 2^-6 steps: all of a sum's bits are within 2^4 .. 2^-18
    x = a[:, 5:6].double() * b[:, 5].double() + bias.double()
    assert torch.equal(x.float().double(), x) and -11.5 <= x.min() and x.max() <= 12.625
    got = sam_hip.mx_matmul(*sam_hip.mx_pack(a.cuda()), *sam_hip.mx_pack(b.cuda()), bias.cuda(), gelu=True, dtype=dt)
    check(got, x, dt)
