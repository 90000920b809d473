"""The paged memory in 4 bits on an MI355X: kv_write and kv_read bit for bit the definition's codes, scales and values, and
paged_attention over them within the bounds that test_paged_attention_gpu.py derives."""
import pytest
import torch

import mx_ref
import paged_ref as ref
from test_kv_cache_gpu import tables
from test_paged_attention_gpu import DT, P_UNIT, Case

pytestmark = pytest.mark.gpu
E2M1 = torch.float4_e2m1fn_x2


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


def pool(pages, heads, page, d, seed=0, scales=(124, 128)):
    """A pool of any codes, with scales that keep attention's scores moderate."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda", dtype=torch.uint8)
    k, v = (rnd(0, 255, pages, heads, page, d // 2).view(E2M1) for _ in range(2))
    return k, v, rnd(*scales, pages, heads, page, d // 32), rnd(*scales, pages, heads, page, d // 32)


class Case4(Case):
    def __init__(self, chunks, lens, hkv, g, d, page, dtype, seed=0, spare=3):
        super().__init__(chunks, lens, hkv, g, d, page, dtype, False, seed, spare)
        self.k, self.v, self.ks, self.vs = pool(self.k.shape[0], hkv, page, d, seed)

    def held(self):
        return tuple(mx_ref.values(x, s).to(DT[self.dtype]) for x, s in ((self.k, self.ks), (self.v, self.vs)))


CASES = [  # chunks, lens, heads, page, d
    ([1], [1], 1, 16, 64), ([5, 0, 3], [5, 7, 40], 3, 8, 96), ([130], [577], 2, 24, 128), ([1] * 70, list(range(1, 71)), 2, 16, 64),
    ([40, 9], [40, 100], 1, 100, 256), ([3, 3, 3], [3, 5, 64], 5, 1, 32), ([64, 1], [64, 65], 4, 64, 160), ([7], [7], 7, 256, 224)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_write_then_read(hip, dtype, case):
    chunks, lens, heads, page, d = case
    dt, t = DT[dtype], sum(chunks)
    width = -(-max(lens) // page) + 1
    pages = sum(-(-n // page) for n in lens) + 4
    table, starts = tables(chunks, lens, page, width, pages)
    kp, vp, ks, vs = pool(pages, heads, page, d, 7, (0, 256))
    before = [x.clone() for x in (kp, vp, ks, vs)]
    g = torch.Generator(device="cuda").manual_seed(1)
    k = (torch.randn(t, heads, d, generator=g, device="cuda") * torch.pow(10.0, torch.randint(-2, 3, (t, heads, 1), generator=g, device="cuda").float())).to(dt)
    v = torch.randn(t, heads, d, generator=g, device="cuda").to(dt)
    v[0, 0] = 0
    ti, si, li = table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    assert hip.kv_write(k, v, kp, vp, ti, si, li, ks, vs) is None
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for new, p, s in ((k, kp, ks), (v, vp, vs)):
        _, codes, exps = mx_ref.quantise(new.cpu())
        for b in range(len(lens)):
            for i, at in enumerate(ref.positions(starts, lens, b)):
                pg, slot = int(table[b, at // page]), at % page
                touched[pg, slot] = True
                assert torch.equal(p.cpu().view(torch.uint8)[pg, :, slot], mx_ref.packed(codes[starts[b] + i]))
                assert torch.equal(s.cpu()[pg, :, slot], exps[starts[b] + i])
    for x, old in zip((kp, vp, ks, vs), before):
        a, o = x.cpu().view(torch.uint8).transpose(1, 2), old.cpu().view(torch.uint8).transpose(1, 2)
        assert torch.equal(a[~touched], o[~touched])
    for out_dt in DT.values():
        for max_len in (max(lens), max(lens) + 3, max(1, max(lens) // 2), 0):
            rk, rv = hip.kv_read(kp, vp, ti, li, max_len, ks, vs, dtype=out_dt)
            assert rk.dtype == out_dt and rk.shape == (len(lens), max_len, heads, d)
            for r, p, s in ((rk, kp, ks), (rv, vp, vs)):
                held = mx_ref.values(p, s)
                want = torch.zeros(len(lens), max_len, heads, d, dtype=torch.float64)
                for b, n in enumerate(lens):
                    rows, _ = ref.gather(held, table, b, min(n, max_len), page)
                    want[b, : len(rows)] = rows
                assert torch.equal(torch.nan_to_num(r.cpu().double(), 9e99, 8e99, -8e99),
                                   torch.nan_to_num(want.to(out_dt).double(), 9e99, 8e99, -8e99))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_row_is_held_as_mx_pack_holds_it(hip, dtype):
    """Ties, subnormals, the largest values, blocks that are not finite beside others that are."""
    f = torch.finfo(DT[dtype])
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 0.0, -0.0, 1e-6, 4.5, 3.0, 2.0] * 2).double()
    blocks = [ties, ties * 2.0 ** -14, ties * (1 + 2 * f.eps), torch.full((32,), f.max).double(), torch.full((32,), f.tiny).double(),
              torch.full((32,), f.smallest_normal * f.eps).double(), torch.zeros(32).double(), torch.cat([torch.tensor([float("nan")]), torch.ones(31)]).double(),
              torch.cat([torch.ones(31), torch.tensor([-float("inf")])]).double(), torch.ones(32).double()]
    x = torch.stack([torch.cat([blocks[(i + j) % 10] for j in range(8)]) for i in range(10)]).to(DT[dtype]).cuda().view(10, 1, 256)
    kp, vp, ks, vs = pool(1, 1, 10, 256)
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    hip.kv_write(x, x.flip(0).contiguous(), kp, vp, i(0).view(1, 1), i(0, 10), i(10), ks, vs)
    codes, scale = hip.mx_pack(x[:, 0])
    assert torch.equal(kp[0, 0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(ks[0, 0], scale)
    assert torch.equal(vp[0, 0].view(torch.uint8), codes.view(torch.uint8).flip(0)) and torch.equal(vs[0, 0], scale.flip(0))


SHAPES = [  # chunks, lens, key heads, group, d, page
    ([1], [1], 1, 1, 64, 16), ([1], [577], 8, 1, 64, 16), ([1, 1, 1], [63, 64, 65], 2, 4, 128, 16),
    ([5, 0, 17], [5, 9, 130], 2, 3, 96, 24), ([33], [33], 1, 2, 256, 8), ([40, 3], [300, 3], 1, 1, 256, 64),
    ([100, 7, 64], [100, 200, 64], 2, 5, 96, 100), ([70], [70], 3, 1, 32, 1), ([130], [389], 1, 8, 128, 32),
    ([1, 2], [1000, 700], 1, 8, 128, 64), ([2], [2], 1, 16, 32, 16), ([65], [200], 2, 2, 64, 7), ([1], [3000], 1, 7, 128, 128),
    ([16, 16], [400, 17], 2, 1, 256, 16), ([3], [129], 1, 1, 160, 16), ([20], [150], 1, 2, 192, 32), ([200], [260], 1, 1, 64, 16),
    ([70, 40], [150, 64], 2, 1, 160, 16), ([90], [200], 1, 1, 224, 16), ([80], [80], 1, 1, 32, 8), ([1], [90], 2, 1, 224, 16)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_the_definition(hip, dtype, shape):
    c = Case4(*shape, dtype, spare=0 if shape[4] % 64 else 3)
    for causal in (True, False):
        c.check(c.run(hip, causal), causal)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("max_q, max_len", [(1, 1), (1, 4000), (500, 64), (64, 1 << 16), (0, 0)])
def test_hints_shape_the_launch_alone(hip, dtype, max_q, max_len):
    for shape in (([100, 7, 1], [100, 200, 300], 2, 3, 128, 16), ([9], [700], 1, 1, 64, 16), ([30], [90], 1, 4, 256, 16)):
        c = Case4(*shape, dtype)
        c.check(c.run(hip, True, max_q=max_q, max_len=max_len), True)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("chunks, lens, hkv, g, d", [
    ([300, 260, 7], [5000, 2600, 300], 1, 1, 64), ([40], [2100], 1, 1, 256), ([3, 1], [30000, 600], 1, 2, 64), ([1], [70000], 2, 4, 128)])
def test_split_keys(hip, dtype, chunks, lens, hkv, g, d):
    if dtype == "f32" and max(chunks) > 100:
        chunks = [3 for _ in chunks]
    c = Case4(chunks, lens, hkv, g, d, 16, dtype)
    c.check(c.run(hip, True, max_q=max(chunks), max_len=max(lens)), True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_see_nothing_are_zero(hip, dtype, d):
    for chunks, lens in (([4, 3], [0, 5]), ([40], [3]), ([7, 2], [-4, 2])):
        c = Case4(chunks, lens, 2, 2, d, 16, dtype)
        for causal in (True, False):
            got = c.run(hip, causal)
            c.check(got, causal)
            if lens[0] <= 0:
                assert (got[: chunks[0]] == 0).all()
    c = Case4([5, 20], [70, 50], 2, 2, d, 16, dtype)
    c.table[0, 1], c.table[0, 3], c.table[1, :] = 1 << 20, -7, -1
    c.ti = c.table.cuda()
    got = c.run(hip, True)
    c.check(got, True)
    assert (got[5:] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("chunk", [3, 60, 200])
def test_nan_blocks_stay_with_the_rows_that_see_them(hip, dtype, d, chunk):
    """Scale bytes of 255: past the end and in pages of nobody they reach no row; at a position, the rows behind it alone, a
    value's in its own block's columns. Infinities of f16 (large scales) likewise."""
    lens = [chunk + 90]
    c = Case4([chunk], lens, 1, 2, d, 16, dtype)
    clean = c.run(hip, True)
    used = set(c.table.flatten().tolist())
    for page in range(c.k.shape[0]):
        if page not in used:
            c.ks[page], c.vs[page] = 255, 255
    last = int(c.table[0, (lens[0] - 1) // 16])
    c.ks[last, :, (lens[0] - 1) % 16 + 1:], c.vs[last, :, (lens[0] - 1) % 16 + 1:] = 255, 255
    assert torch.equal(c.run(hip, True), clean)
    for i, byte in enumerate((255, 254)):
        for into in ("v", "k"):
            at = lens[0] - chunk + chunk // 2 - i  # a position inside the chunk
            t = Case4([chunk], lens, 1, 2, d, 16, dtype)
            getattr(t, into + "s")[int(t.table[0, at // 16]), 0, at % 16, d // 64] = byte
            got = t.run(hip, True)
            row = at - (lens[0] - chunk)  # the first row that sees it
            assert torch.isfinite(got[:row]).all()
            k, v = t.held()
            want, bound = ref.attention(t.q[:row].cpu(), k, v, t.table, [0, row], [at], d ** -0.5, True, P_UNIT[dtype])
            assert ((got[:row].cpu().double() - want).abs() <= ref.with_rounding(bound, want, DT[dtype])).all()
            lo = d // 64 * 32
            if into == "v":
                assert torch.isfinite(got[..., :lo]).all() and torch.isfinite(got[..., lo + 32:]).all()
                if byte == 255:
                    assert torch.isnan(got[row:, :, lo:lo + 32]).all()
            elif byte == 255:
                assert torch.isnan(got[row:]).all()


def test_shared_pages_strides_and_in_place(hip):
    c = Case4([30, 4], [80, 20], 2, 2, 64, 16, "f16")
    want = c.run(hip, True)
    packed = torch.zeros(34, 3, 4, 64, device="cuda", dtype=torch.float16)
    packed[:, 1] = c.q
    assert torch.equal(c.run(hip, True, q=packed[:, 1]), want)
    out = torch.zeros(34, 3, 4, 64, device="cuda", dtype=torch.float16)
    assert torch.equal(c.run(hip, True, out=out[:, 2]), want) and (out[:, :2] == 0).all()
    assert torch.equal(c.run(hip, True, out=c.q), want)
    c = Case4([1, 1], [100, 100], 2, 2, 128, 16, "bf16")
    c.table[1] = c.table[0]
    c.table[0, 3] = c.table[0, 2]
    c.table[1, 3] = c.table[0, 3]
    c.ti = c.table.cuda()
    c.q[1] = c.q[0]
    got = c.run(hip, True)
    assert torch.equal(got[0], got[1])
    c.check(got, True)


@pytest.mark.parametrize("chunk", [1, 50])
def test_pages_past_4_gib(hip, chunk):
    """Pools of more than 2^32 bytes and 2^33 values, whose last pages are written, read and attended."""
    pages, heads, page, d = 72000, 8, 128, 128
    kp, vp = (torch.zeros(pages, heads, page, d // 2, device="cuda", dtype=torch.uint8).view(E2M1) for _ in range(2))
    ks, vs = (torch.full((pages, heads, page, d // 32), 127, device="cuda", dtype=torch.uint8) for _ in range(2))
    assert kp.numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    n = 200
    k, v, q = rnd(n, heads, d), rnd(n, heads, d), rnd(chunk, heads, d)
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    far, near = i(pages - 1, pages - 2).view(1, 2), i(0, 1).view(1, 2)
    out = []
    for table in (far, near):
        hip.kv_write(k, v, kp, vp, table, i(0, n), i(n), ks, vs)
        out.append((*hip.kv_read(kp, vp, table, i(n), n, ks, vs, dtype=torch.float16),
                    hip.paged_attention(q, kp, vp, table, i(0, chunk), i(n), ks, vs, max_len=n)))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert torch.equal(out[0][0][0], mx_ref.quantise(k.cpu())[0].half().cuda())


def test_a_captured_step_replays(hip):
    """A decoding step (write and attend) as a graph, replayed with eager work in between, against the eager results."""
    c = Case4([1, 1, 1], [40, 300, 129], 2, 4, 128, 16, "bf16")
    k, v = torch.randn(3, 2, 128, device="cuda").bfloat16(), torch.randn(3, 2, 128, device="cuda").bfloat16()
    other = [x.clone() for x in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.ks, c.vs)]
    eager_pool = lambda: (other[0].view(E2M1), other[1].view(E2M1), c.ti, c.si, c.li, other[2], other[3])

    def step(kp, vp, ti, si, li, ks, vs):
        hip.kv_write(k, v, kp, vp, ti, si, li, ks, vs)
        return hip.paged_attention(c.q, kp, vp, ti, si, li, ks, vs, max_q=1, max_len=310)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c.k, c.v, c.ti, c.si, c.li, c.ks, c.vs)
    for i in range(4):
        c.q.copy_(torch.randn_like(c.q))
        k.copy_(torch.randn_like(k))
        graph.replay()
        want = step(*eager_pool())
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        c.li += 1
        c.li.clamp_(max=c.ti.shape[1] * 16)


def test_refusals(hip):
    c = Case4([4], [20], 2, 2, 64, 16, "f16")
    k = torch.zeros(4, 2, 64, device="cuda", dtype=torch.float16)
    k80 = torch.zeros(4, 2, 80, device="cuda", dtype=torch.float16)
    p80 = torch.zeros(3, 2, 16, 40, device="cuda", dtype=torch.uint8).view(E2M1)
    s80 = torch.zeros(3, 2, 16, 3, device="cuda", dtype=torch.uint8)
    for call in (lambda: hip.kv_write(k, k, c.k, c.v, c.ti, c.si, c.li), lambda: hip.kv_write(k, k, c.k, c.v, c.ti, c.si, c.li, c.ks[..., 0], c.vs[..., 0]),
                 lambda: hip.kv_write(k, k, c.k.view(torch.uint8), c.v.view(torch.uint8), c.ti, c.si, c.li, c.ks, c.vs),
                 lambda: hip.kv_write(k[..., :32], k[..., :32], c.k, c.v, c.ti, c.si, c.li, c.ks, c.vs),
                 lambda: hip.kv_write(k80, k80, p80, p80, c.ti, c.si, c.li, s80, s80), lambda: hip.kv_read(c.k, c.v, c.ti, c.li, 4, c.ks, c.vs),
                 lambda: hip.kv_read(c.k, c.v, c.ti, c.li, 4, c.ks.transpose(0, 1).contiguous().transpose(0, 1), c.vs, dtype=torch.float16),
                 lambda: hip.paged_attention(c.q, c.k, c.v, c.ti, c.si, c.li), lambda: c.run(hip, True, q=c.q[..., :32])):
        with pytest.raises(hip.SamHipError):
            call()
