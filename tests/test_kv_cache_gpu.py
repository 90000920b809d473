"""kv_write and kv_read on an MI355X: bit for bit the definition's values (a power-of-two scale leaves the rounding to
e4m3 as the only one), in their places, with everything else in the pool untouched."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


def pool(pages, heads, page, d, dtype, fp8, seed=0):
    """A pool filled with a pattern that a stray write would change."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages, heads, page, d)
    if fp8:
        k, v = (torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
                for _ in range(2))
        ks, vs = (torch.randint(100, 150, shape[:3], generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
        return k, v, ks, vs
    return (*(torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2)), None, None)


def tables(chunks, lens, page, width, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(-(-min(max(n, 0), width * page) // page)):
            table[b, j] = order.pop()
    starts = [sum(chunks[:i]) for i in range(len(chunks) + 1)]
    return table, starts


def values(p, s):
    return p.cpu().double() if s is None else p.cpu().float().double() * torch.pow(torch.tensor(2.0, dtype=torch.float64), s.cpu().double() - 127)[..., None]


CASES = [  # chunks, lens, heads, page, d
    ([1], [1], 1, 16, 64), ([5, 0, 3], [5, 7, 40], 3, 8, 80), ([130], [577], 2, 24, 128), ([1] * 70, list(range(1, 71)), 2, 16, 64),
    ([40, 9], [40, 100], 1, 100, 256), ([3, 3, 3], [3, 5, 64], 5, 1, 72), ([64, 1], [64, 65], 4, 64, 8), ([7], [7], 7, 256, 96)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_write_then_read(hip, dtype, fp8, case):
    chunks, lens, heads, page, d = case
    dt, t = DT[dtype], sum(chunks)
    width = -(-max(lens) // page) + 1
    pages = sum(-(-n // page) for n in lens) + 4
    table, starts = tables(chunks, lens, page, width, pages)
    kp, vp, ks, vs = pool(pages, heads, page, d, dt, fp8)
    before = [x.clone() for x in (kp, vp, ks, vs) if x is not None]
    g = torch.Generator(device="cuda").manual_seed(1)
    k = (torch.randn(t, heads, d, generator=g, device="cuda") * torch.pow(10.0, torch.randint(-2, 3, (t, heads, 1), generator=g, device="cuda").float())).to(dt)
    v = torch.randn(t, heads, d, generator=g, device="cuda").to(dt)
    v[0, 0] = 0
    ti, si, li = table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    assert hip.kv_write(k, v, kp, vp, ti, si, li, ks, vs) is None
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for new, p, s in ((k, kp, ks), (v, vp, vs)):
        want, exps = ref.quantise(new.cpu()) if fp8 else (new.cpu().double(), None)
        got = values(p, s)
        for b in range(len(lens)):
            for i, at in enumerate(ref.positions(starts, lens, b)):
                pg, slot = int(table[b, at // page]), at % page
                touched[pg, slot] = True
                assert torch.equal(got[pg, :, slot], want[starts[b] + i])
                if fp8:
                    assert torch.equal(s.cpu()[pg, :, slot], exps[starts[b] + i])
    free = ~touched
    for x, old in zip([x for x in (kp, vp, ks, vs) if x is not None], before):
        a, o = x.cpu().view(torch.uint8).reshape(pages, heads, page, -1), old.cpu().view(torch.uint8).reshape(pages, heads, page, -1)
        assert torch.equal(a.transpose(1, 2)[free], o.transpose(1, 2)[free])
    for out_dt in ([torch.float32, torch.float16, torch.bfloat16] if fp8 else [dt]):
        for max_len in (max(lens), max(lens) + 3, max(1, max(lens) // 2), 0):
            rk, rv = hip.kv_read(kp, vp, ti, li, max_len, ks, vs, dtype=out_dt)
            assert rk.dtype == out_dt and rk.shape == (len(lens), max_len, heads, d)
            for r, p, s in ((rk, kp, ks), (rv, vp, vs)):
                held = values(p, s)
                want = torch.zeros(len(lens), max_len, heads, d, dtype=torch.float64)
                for b, n in enumerate(lens):
                    rows, _ = ref.gather(held, table, b, min(n, max_len), page)
                    want[b, : len(rows)] = rows
                assert torch.equal(r.cpu(), want.to(out_dt))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_every_rounding_and_extreme_rows(hip, dtype):
    """Rows of ties, subnormal codes, the largest and smallest scales, values that are not finite."""
    dt = DT[dtype]
    d = 64
    f = torch.finfo(dt)
    rows = [torch.linspace(-448, 448, d), torch.linspace(-1, 1, d) * 2.0 ** -6, torch.full((d,), f.max), torch.full((d,), f.tiny),
            torch.full((d,), f.smallest_normal * f.eps), torch.zeros(d), torch.tensor([448.0, 449.0] * 32), torch.tensor([450.0] + [1e-3] * 63),
            torch.tensor([float("inf"), 1.0, float("nan"), -float("inf")] * 16), torch.tensor([float("nan")] * 64)]
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    grid = torch.unique(codes[torch.isfinite(codes)])
    mids = torch.cat([(grid[1:] + grid[:-1]) / 2, torch.tensor([448.0] * 3)])  # ties
    rows += [torch.cat([m, torch.full((d - len(m),), 448.0)]) for m in mids.split(d - 1)]
    x = torch.stack(rows).to(dt).cuda().view(len(rows), 1, d)
    kp, vp, ks, vs = pool(1, 1, len(rows), d, dt, True)
    one = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    hip.kv_write(x, x.flip(0).contiguous(), kp, vp, one(0).view(1, 1), one(0, len(rows)), one(len(rows)), ks, vs)
    want, exps = ref.quantise(x.cpu())
    assert torch.equal(ks.cpu()[0], exps.view(1, -1)) and torch.equal(vs.cpu()[0], exps.flip(0).view(1, -1))
    got = values(kp, ks)[0, 0]
    assert torch.equal(torch.isnan(got), torch.isnan(want[:, 0])) and torch.equal(got.nan_to_num(), want[:, 0].nan_to_num())


def test_strides_views_and_a_second_write(hip):
    g = torch.Generator(device="cuda").manual_seed(3)
    packed = torch.randn(9, 3, 2, 64, generator=g, device="cuda").half()
    table, starts, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[2, 0], [1, 3]], [0, 4, 9], [20, 9]))
    for k, v in ((packed[:, 0], packed[:, 1]), (packed[:, 1].transpose(1, 2).contiguous().transpose(1, 2), packed[:, 2]),
                 (torch.empty(9 * 128 + 1, device="cuda", dtype=torch.float16)[1:].view(9, 2, 64).copy_(packed[:, 0]), packed[:, 1])):
        a, b = pool(4, 2, 16, 64, torch.float16, False), pool(4, 2, 16, 64, torch.float16, False)
        hip.kv_write(k, v, a[0], a[1], table, starts, lens)
        hip.kv_write(k.contiguous(), v.contiguous(), b[0], b[1], table, starts, lens)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        rk, rv = hip.kv_read(a[0], a[1], table, lens, 20)
        assert torch.equal(rk[0, 16:20], k[:4]) and torch.equal(rv[1, 4:9], v[4:])


def test_tokens_and_pages_outside_are_left_alone(hip):
    """Negative positions, positions past the table, page entries that name nothing, tokens behind the last sequence."""
    k = torch.ones(12, 1, 64, device="cuda", dtype=torch.float16)
    kp, vp, _, _ = pool(3, 1, 4, 64, torch.float16, False)
    old = kp.clone()
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    hip.kv_write(k, k, kp, vp, i([[7, -1], [3, 1 << 30]]), i([0, 4, 8]), i([8, 8]))
    hip.kv_write(k, k, kp, vp, i([[0, 1], [2, -5]]), i([0, 4, 8]), i([-3, 0]))  # before position 0
    hip.kv_write(k, k, kp, vp, i([[0, 1], [2, -5]]), i([0, 4, 8]), i([1 << 30, 2 ** 31 - 1]))  # past the table
    hip.kv_write(k, k, kp, vp, i([[0, 1]]), i([12, 12]), i([4]))  # no tokens of any sequence
    hip.kv_write(k[:0], k[:0], kp, vp, i([[0, 1]]), i([0, 0]), i([4]))
    assert torch.equal(kp, old)
    hip.kv_write(k, k, kp, vp, i([[0, 1], [2, -5]]), i([2, 4, 10]), i([1, 6]))  # one of 2 fits; 4 of 6 have a page
    got = kp[:, 0, :, 0] == 1
    assert got.tolist() == [[True, False, False, False], [False] * 4, [True] * 4]
    rk, _ = hip.kv_read(kp, vp, i([[2, 7], [0, -1]]), i([8, -2]), 9)
    assert (rk[0, :4] == 1).all() and (rk[0, 4:] == 0).all() and (rk[1] == 0).all()


def test_refusals(hip):
    k = torch.zeros(2, 1, 64, device="cuda", dtype=torch.float16)
    kp, vp, _, _ = pool(3, 1, 4, 64, torch.float16, False)
    k8, v8, ks, vs = pool(3, 1, 4, 64, torch.float16, True)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    t, s, n = i([[0, 1]]), i([0, 2]), i([2])
    for call in (lambda: hip.kv_write(k.float(), k.float(), kp, vp, t, s, n), lambda: hip.kv_write(k, k, kp, vp, t.long(), s, n),
                 lambda: hip.kv_write(k, k, kp, vp, t, s[:1], n), lambda: hip.kv_write(k, k, kp, vp, t, s, n.long()),
                 lambda: hip.kv_write(k, k[:1], kp, vp, t, s, n), lambda: hip.kv_write(k, k, k8, v8, t, s, n),
                 lambda: hip.kv_write(k, k, kp, vp, t, s, n, ks, vs), lambda: hip.kv_write(k, k, k8, v8, t, s, n, ks[:, :, :3], vs),
                 lambda: hip.kv_write(k, k, kp.transpose(1, 2), vp.transpose(1, 2), t, s, n), lambda: hip.kv_write(k, k, kp, v8, t, s, n),
                 lambda: hip.kv_read(k8, v8, t, n, 4, ks, vs), lambda: hip.kv_read(kp, vp, t, n, -1),
                 lambda: hip.kv_read(kp, vp, t, n, 4, dtype=torch.float32), lambda: hip.kv_write(k, k, kp, vp, t, s.cpu(), n)):
        with pytest.raises(hip.SamHipError):
            call()
