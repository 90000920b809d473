"""4-bit numbers on an MI355X: packing and unpacking bit for bit, products and linear layers within their f32 sums'
roundings."""
import pytest
import torch

import mx_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


def randn(*shape, dtype=torch.float32, seed=0, spread=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    if spread:
        x = x * torch.pow(10.0, torch.randint(-spread, spread + 1, (*shape[:-1], 1), generator=g, device="cuda").float())
    return x.to(dtype)


def same(got, want):
    """Equal values, NaN in the same places."""
    got, want = got.cpu().double(), want.double()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0, 9e99, -9e99), want.nan_to_num(0, 9e99, -9e99))


def check_pack(hip, x, outs=("f32", "f16", "bf16")):
    codes, scale = hip.mx_pack(x)
    assert codes.dtype == torch.float4_e2m1fn_x2 and codes.shape == (*x.shape[:-1], x.shape[-1] // 2)
    assert scale.dtype == torch.uint8 and scale.shape == (*x.shape[:-1], x.shape[-1] // 32)
    value, want, exps = ref.quantise(x.cpu())
    assert torch.equal(scale.cpu(), exps)
    assert torch.equal(codes.cpu().view(torch.uint8), ref.packed(want))
    for o in outs:
        back = hip.mx_unpack(codes, scale, DT[o])
        assert back.dtype == DT[o] and back.shape == x.shape
        assert same(back, value.to(DT[o]).double())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(32,), (1, 64), (3, 5, 96), (7, 1280), (196, 1024), (600, 4096), (2, 0, 64)])
def test_pack_and_unpack(hip, dtype, shape):
    check_pack(hip, randn(*shape, dtype=DT[dtype], spread=2))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_every_rounding_and_extreme_blocks(hip, dtype):
    """Ties, values next to them, subnormals, the largest and smallest scales, zeros of both signs, values not finite."""
    dt = DT[dtype]
    f = torch.finfo(dt)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.cat([ties, ties * (1 + 2 * f.eps), ties * (1 - 2 * f.eps), torch.tensor([6.0, -6.0, 0.0, -0.0, -0.25, -2.5, 1e-6, -1e-6, 4.0, 3.0, 0.5])])
    rows = [near, near * 2.0 ** -14, near * 2.0 ** 10, torch.full((32,), f.max), torch.full((32,), f.tiny), torch.full((32,), f.smallest_normal * f.eps),
            torch.zeros(32), -torch.zeros(32), torch.cat([torch.tensor([f.max]), torch.full((31,), f.tiny)]), torch.linspace(-6, 6, 32),
            torch.tensor([6.0] * 31 + [6.0 * (1 + 2 * f.eps)]), torch.cat([torch.tensor([float("inf")]), torch.ones(31)]),
            torch.cat([torch.ones(31), torch.tensor([float("nan")])]), torch.full((32,), -float("inf")), torch.ones(32)]
    check_pack(hip, torch.stack([r.double().to(dt) for r in rows]).cuda())
    check_pack(hip, torch.cat([r.double().to(dt) for r in rows]).cuda())  # one row: blocks do not reach one another


def test_every_code_and_scale_unpacks(hip):
    codes = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(1, 256, 16).expand(256, 256, 16).contiguous()
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 256, 1).contiguous()
    want = ref.values(codes, scale)
    for dt in DT.values():
        got = hip.mx_unpack(codes.cuda().view(torch.float4_e2m1fn_x2), scale.cuda(), dt)
        assert same(got, want.to(dt).double())


def operands(m, n, k, dtype, seed, spread=1):
    a, b = randn(m, k, seed=seed, spread=spread), randn(n, k, seed=seed + 1) * k ** -0.5
    return a.to(dtype), b.to(dtype), randn(n, dtype=dtype, seed=seed + 2)


SIZES = [(1, 1, 32), (1, 16, 32), (3, 5, 64), (7, 1280, 5120), (16, 16, 128), (17, 33, 96), (32, 100, 160), (1, 4099, 1024), (33, 64, 128), (64, 64, 4096),
         (65, 130, 224), (200, 129, 384), (128, 128, 32), (300, 260, 1280), (1, 7, 8192), (1601, 2001, 96), (1700, 1930, 128), (2100, 1600, 416), (577, 36, 768)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", SIZES)
def test_products(hip, dtype, size):
    m, n, k = size
    dt = DT[dtype]
    a, b, bias = operands(m, n, k, dt, m + n + k)
    (ac, asc), (bc, bsc) = hip.mx_pack(a), hip.mx_pack(b)
    av, bv = ref.values(ac, asc), ref.values(bc, bsc)
    for with_bias, act in ((False, False), (True, False), (True, True), (False, True)):
        got = hip.mx_matmul(ac, asc, bc, bsc, bias if with_bias else None, gelu=act, dtype=dt)
        assert got.shape == (m, n) and got.dtype == dt
        want, bound = ref.product(av, bv, bias.cpu() if with_bias else None, act, dt)
        assert ((got.cpu().double() - want).abs() <= bound).all(), (with_bias, act, float(((got.cpu().double() - want).abs() / bound).max()))
        assert torch.equal(hip.mx_linear(a, bc, bsc, bias if with_bias else None, gelu=act), got)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [(8, 4100, 64), (9, 4100, 32), (9, 5120, 1280), (12, 5003, 96), (16, 6144, 544), (17, 8189, 160), (32, 4600, 1120), (16, 8192, 4096)])
def test_few_rows_of_wide_layers(hip, dtype, size):
    """Two blocks of columns a workgroup, ragged ones too, with scales that begin at any byte."""
    m, n, k = size
    dt = DT[dtype]
    a, b, bias = operands(m, n, k, dt, m + n + k)
    (ac, asc), (bc, bsc) = hip.mx_pack(a), hip.mx_pack(b)
    want, bound = ref.product(ref.values(ac, asc), ref.values(bc, bsc), bias.cpu(), True, dt)
    off = [torch.full((s.numel() + 3,), 255, device="cuda", dtype=torch.uint8)[i:i + s.numel()].view(s.shape).copy_(s) for i, s in ((1, asc), (3, bsc))]
    for sa, sb in ((asc, bsc), off):
        got = hip.mx_matmul(ac, sa, bc, sb, bias, gelu=True, dtype=dt)
        assert ((got.cpu().double() - want).abs() <= bound).all(), float(((got.cpu().double() - want).abs() / bound).max())
        assert torch.equal(hip.mx_linear(a, bc, sb, bias, gelu=True), got)


@pytest.mark.parametrize("m", [1, 20, 100, 1601])
def test_nan_blocks_stay_in_their_rows_and_columns(hip, m):
    n, k = 2001 if m > 1000 else 90, 160
    a, b, _ = operands(m, n, k, torch.float16, 5)
    a[m // 2, 40], b[n // 3, 159] = float("nan"), -float("inf")
    got = hip.mx_linear(a, *hip.mx_pack(b))
    clean = hip.mx_linear(a.nan_to_num(0.0), *hip.mx_pack(b.nan_to_num(0.0, 0.0, 0.0)))
    nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    nan[m // 2], nan[:, n // 3] = True, True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], clean[~nan])


def test_scales_at_both_ends(hip):
    """2^-126 by 2^126 blocks: the products are ordinary numbers."""
    one = torch.ones(40, 64, device="cuda")
    a, b = one * 2.0 ** -124, one * 2.0 ** 125
    got = hip.mx_matmul(*hip.mx_pack(a), *hip.mx_pack(b))
    assert torch.equal(got, torch.full((40, 40), 128.0, device="cuda"))
    assert torch.isinf(hip.mx_matmul(*hip.mx_pack(b), *hip.mx_pack(b))).all()


def test_views_leading_dimensions_and_alignment(hip):
    x = randn(2, 3, 50, 96, dtype=torch.float16)
    w = randn(70, 96, dtype=torch.float16, seed=1)
    wc, ws = hip.mx_pack(w)
    want = hip.mx_linear(x.reshape(300, 96), wc, ws)
    assert torch.equal(hip.mx_linear(x, wc, ws).view(300, 70), want)
    assert torch.equal(hip.mx_linear(x.transpose(1, 2), wc, ws), want.view(2, 3, 50, 70).transpose(1, 2))
    off = torch.empty(300 * 96 + 1, device="cuda", dtype=torch.float16)[1:].view(300, 96).copy_(x.view(300, 96))
    assert torch.equal(hip.mx_linear(off, wc, ws), want)
    # scales off a 4-byte boundary where k would allow dwords
    x, w = randn(100, 256, dtype=torch.bfloat16), randn(100, 256, dtype=torch.bfloat16, seed=1)
    (xc, xs), (wc, ws) = hip.mx_pack(x), hip.mx_pack(w)
    shifted = torch.empty(801, device="cuda", dtype=torch.uint8)[1:].view(100, 8).copy_(ws)
    codes = torch.empty(100 * 128 + 1, device="cuda", dtype=torch.uint8)[1:].view(100, 128).copy_(wc.view(torch.uint8)).view(torch.float4_e2m1fn_x2)
    assert torch.equal(hip.mx_matmul(xc, xs, codes, shifted), hip.mx_matmul(xc, xs, wc, ws))
    assert hip.mx_matmul(xc[:0], xs[:0], wc, ws).shape == (0, 100) and hip.mx_matmul(xc, xs, wc[:0], ws[:0]).shape == (100, 0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 16, 17])
def test_the_workspace_size_and_extreme_rows(hip, dtype, m):
    """A layer on rows that it packs on the way, and with a workspace, against packing them first: blocks of zeros, of the
    largest and smallest values, of values that are not finite."""
    f = torch.finfo(DT[dtype])
    x, w = randn(m, 320, dtype=DT[dtype], seed=m), randn(50, 320, dtype=DT[dtype], seed=1)
    x[0, :32], x[0, 32:64], x[0, 64:96], x[m // 2, 96:128], x[m - 1, 128:160] = 0, f.tiny, -0.0, f.smallest_normal * f.eps, 2.0 ** 10
    wc, ws = hip.mx_pack(w)
    assert hip.load().sam_hip_mx_linear_workspace_size(m, 50, 320) == (0 if m <= 16 else m * 170)
    assert torch.equal(hip.mx_linear(x, wc, ws), hip.mx_matmul(*hip.mx_pack(x), wc, ws, dtype=DT[dtype]))
    x[m - 1, 300], x[0, 10] = float("inf"), float("nan")
    got = hip.mx_linear(x, wc, ws)
    assert torch.isnan(got[0]).all() and torch.isnan(got[m - 1]).all() and (m < 3 or torch.isfinite(got[1:m - 1]).all())


def test_rows_behind_the_result_are_left_alone(hip):
    """A result of odd sizes inside a larger allocation: nothing around it changes (through the C entry)."""
    for m, n in ((5, 33), (70, 67), (1601, 2001)):
        a, b, _ = operands(m, n, 96, torch.float16, 3)
        (ac, asc), (bc, bsc) = hip.mx_pack(a), hip.mx_pack(b)
        room = torch.full((m * n + 4096,), 7.0, device="cuda", dtype=torch.float16)
        rc = hip.load().sam_hip_mx_matmul(ac.data_ptr(), asc.data_ptr(), bc.data_ptr(), bsc.data_ptr(), None, room[2048:].data_ptr(), 1, m, n, 96, 0, hip._stream())
        assert rc == 0
        assert torch.equal(room[2048:2048 + m * n].view(m, n), hip.mx_matmul(ac, asc, bc, bsc, dtype=torch.float16))
        assert (room[:2048] == 7).all() and (room[2048 + m * n:] == 7).all()


def test_streams_graphs_and_repeats(hip):
    """Two streams at once, and a captured linear layer replayed on new inputs, with eager work in between, give the eager
    results' bits."""
    w, bias = randn(640, 512, dtype=torch.float16, seed=1), randn(640, dtype=torch.float16, seed=2)
    wc, ws = hip.mx_pack(w)
    xs = [randn(m, 512, dtype=torch.float16, seed=m) for m in (9, 300)]
    want = [hip.mx_linear(x, wc, ws, bias, gelu=True) for x in xs]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(side, xs):
        with torch.cuda.stream(s):
            got.append([hip.mx_linear(x, wc, ws, bias, gelu=True) for _ in range(5)])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(y, b) for y in a)
    static = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [hip.mx_linear(x, wc, ws, bias, gelu=True) for x in static]
    for seed in range(4):
        for x in static:
            x.copy_(randn(*x.shape, dtype=torch.float16, seed=100 + seed))
        graph.replay()
        eager = [hip.mx_linear(x, wc, ws, bias, gelu=True) for x in static]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_refusals(hip):
    x = randn(4, 64, dtype=torch.float16)
    c, s = hip.mx_pack(x)
    bias = randn(4, dtype=torch.float16)
    for call in (lambda: hip.mx_pack(x[:, :40]), lambda: hip.mx_pack(x[:, :0]), lambda: hip.mx_pack(x.double()), lambda: hip.mx_pack(x.cpu()),
                 lambda: hip.mx_pack(x[0, 0]), lambda: hip.mx_unpack(c, s, torch.float64), lambda: hip.mx_unpack(c.view(torch.uint8), s),
                 lambda: hip.mx_unpack(c, s[:, :1]), lambda: hip.mx_unpack(c, s.int()), lambda: hip.mx_matmul(c, s, c[:, :16], s[:, :1]),
                 lambda: hip.mx_matmul(c, s, c[0], s[0]), lambda: hip.mx_matmul(c, s, c, s, bias), lambda: hip.mx_matmul(c, s, c, s, bias[:3], dtype=torch.float16),
                 lambda: hip.mx_matmul(c, s, c, s.cpu()), lambda: hip.mx_linear(x, c, s, bias.float()), lambda: hip.mx_linear(x[:, :32], c, s),
                 lambda: hip.mx_matmul(c, s, c, s, dtype=torch.int32)):
        with pytest.raises(hip.SamHipError):
            call()
    hip.set_enabled(False)
    try:
        for call in (lambda: hip.mx_pack(x), lambda: hip.mx_unpack(c, s), lambda: hip.mx_matmul(c, s, c, s), lambda: hip.mx_linear(x[:0], c, s),
                     lambda: hip.mx_pack(x[:0])):
            with pytest.raises(hip.SamHipDisabled):
                call()
    finally:
        hip.set_enabled(True)
