"""paged_attention on an MI355X against the definition in 64 bits (paged_ref.attention), each element within the bound
of the kernel's roundings: every f32 sum at one rounding a term, P's rounding to the value type, the output's own."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# P beside v: f32 as it is, f16 to half a step of f16, bf16 as two bf16 terms (2^-16)
P_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -16}


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


class Case:
    def __init__(self, chunks, lens, hkv, g, d, page, dtype, fp8, seed=0, spare=3, spread=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed + d + page)
        dt = DT[dtype]
        self.dtype, self.chunks, self.lens, self.page = dtype, chunks, lens, page
        width = max(1, max(-(-n // page) for n in lens))
        pages = sum(-(-max(n, 0) // page) for n in lens) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(lens):
            for j in range(-(-max(n, 0) // page)):
                self.table[b, j] = order.pop()
        self.starts = [sum(chunks[:i]) for i in range(len(chunks) + 1)]
        rnd = lambda *s: torch.randn(s, generator=gen, device="cuda") * spread
        self.q = rnd(self.starts[-1], hkv * g, d).to(dt)
        self.k, self.v = rnd(pages, hkv, page, d).to(dt), rnd(pages, hkv, page, d).to(dt)
        self.ks = self.vs = None
        if fp8:
            e = [torch.randint(121, 126, (pages, hkv, page), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
            self.ks, self.vs = e
            self.k, self.v = ((x.float() * 32).to(torch.float8_e4m3fn) for x in (self.k, self.v))
        self.ti, self.si, self.li = (torch.as_tensor(x, dtype=torch.int32).cuda() for x in (self.table, self.starts, self.lens))

    def held(self):
        if self.ks is None:
            return self.k.cpu(), self.v.cpu()
        two = torch.tensor(2.0, dtype=torch.float64)
        return tuple((x.cpu().float().double() * torch.pow(two, s.cpu().double() - 127)[..., None]).to(DT[self.dtype])
                     for x, s in ((self.k, self.ks), (self.v, self.vs)))

    def run(self, hip, causal, q=None, **kw):
        return hip.paged_attention(self.q if q is None else q, self.k, self.v, self.ti, self.si, self.li, self.ks, self.vs,
                                   causal=causal, **kw)

    def check(self, got, causal, scale=None):
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        k, v = self.held()
        want, bound = ref.attention(self.q.cpu(), k, v, self.table, self.starts, self.lens, scale, causal, P_UNIT[self.dtype])
        bound = ref.with_rounding(bound, want, DT[self.dtype])
        off = (got.cpu().double() - want).abs()
        worst = float((off / bound).max()) if off.numel() else 0.0
        assert worst <= 1.0, f"{worst:.3g} of the bound, {float(off.max()):.3g} off"


SHAPES = [  # chunks, lens, key heads, group, d, page
    ([1], [1], 1, 1, 64, 16), ([1], [577], 8, 1, 64, 16), ([1, 1, 1], [63, 64, 65], 2, 4, 128, 16),
    ([5, 0, 17], [5, 9, 130], 2, 3, 80, 24), ([33], [33], 1, 2, 256, 8), ([40, 3], [300, 3], 1, 1, 256, 64),
    ([100, 7, 64], [100, 200, 64], 2, 5, 96, 100), ([70], [70], 3, 1, 72, 1), ([130], [389], 1, 8, 128, 32),
    ([1, 2], [1000, 700], 1, 8, 128, 64), ([2], [2], 1, 16, 8, 16), ([65], [200], 2, 2, 64, 7), ([1], [3000], 1, 7, 128, 128),
    ([16, 16], [400, 17], 2, 1, 256, 16), ([3], [129], 1, 1, 136, 16), ([20], [150], 1, 2, 200, 32), ([200], [260], 1, 1, 48, 16)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_definition(hip, dtype, fp8, shape):
    c = Case(*shape, dtype, fp8)
    for causal in (True, False):
        c.check(c.run(hip, causal), causal)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("max_q, max_len", [(1, 1), (1, 4000), (500, 64), (64, 1 << 16), (0, 0)])
def test_hints_shape_the_launch_alone(hip, dtype, max_q, max_len):
    """Grids for one row or key, for fewer and for far more than there are, give results within the bound all the same."""
    for shape in (([100, 7, 1], [100, 200, 300], 2, 3, 128, 16), ([9], [700], 1, 1, 64, 16), ([30], [90], 1, 4, 256, 16)):
        c = Case(*shape, dtype, False)
        c.check(c.run(hip, True, max_q=max_q, max_len=max_len), True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_see_nothing_are_zero(hip, dtype, fp8, d):
    """Sequences without keys, more new tokens than the sequence holds, pages that are not there, rows of no sequence."""
    for chunks, lens in (([4, 3], [0, 5]), ([40], [3]), ([7, 2], [-4, 2])):
        c = Case(chunks, lens, 2, 2, d, 16, dtype, fp8)
        for causal in (True, False):
            got = c.run(hip, causal)
            c.check(got, causal)
            if lens[0] <= 0:
                assert (got[: chunks[0]] == 0).all()
    c = Case([5, 20], [70, 50], 2, 2, d, 16, dtype, fp8)
    c.table[0, 1], c.table[0, 3], c.table[1, :] = 1 << 20, -7, -1
    c.ti = c.table.cuda()
    got = c.run(hip, True)
    c.check(got, True)
    assert (got[5:] == 0).all()
    pad = torch.full((40, 4, d), 3.0, device="cuda", dtype=DT[dtype])  # tokens 0..4 and 30..39 belong to no sequence
    q = pad.clone()
    q[5:30] = c.q
    c.si += 5
    for kw in ({}, {"max_len": 1 << 16, "max_q": 1}):
        got = c.run(hip, True, q=q, **kw)
        assert (got[:5] == 0).all() and (got[30:] == 0).all()
        kept = c.run(hip, True, q=q, out=pad.clone(), **kw)
        assert (kept[:5] == 3).all() and (kept[30:] == 3).all() and torch.equal(kept[5:30], got[5:30])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("chunk", [3, 60, 200])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(hip, dtype, fp8, d, chunk):
    """NaN and infinities in keys and values: past the end and in pages of nobody they reach no row; at a position, the
    rows behind it alone, in the value's own column. There an infinity stays one in f32 and f16; in bf16, where P is a
    sum of two terms of either sign (or one of them 0), it may become NaN, as inf - inf and 0 * inf are."""
    lens = [chunk + 90]
    c = Case([chunk], lens, 1, 2, d, 16, dtype, fp8)
    clean = c.run(hip, True)
    bad = [float("nan")] if fp8 else [float("nan"), float("inf"), -float("inf")]
    used = set(c.table.flatten().tolist())

    def put(pages, page, slot, col, x):
        if fp8:
            pages.view(torch.uint8)[page, 0, slot, col] = 0x7F
        else:
            pages[page, 0, slot, col] = x

    for page in range(c.k.shape[0]):
        if page not in used:
            c.k.view(torch.uint8)[page], c.v.view(torch.uint8)[page] = 0x7F, 0x7F
    last = int(c.table[0, (lens[0] - 1) // 16])
    for slot in range((lens[0] - 1) % 16 + 1, 16):
        for col in range(d):
            put(c.k, last, slot, col, bad[0])
            put(c.v, last, slot, col, bad[-1])
    assert torch.equal(c.run(hip, True), clean)
    for i, x in enumerate(bad):
        for into in ("v", "k"):
            at = lens[0] - chunk + chunk // 2 - (i == 1)  # a position inside the chunk
            t = Case([chunk], lens, 1, 2, d, 16, dtype, fp8)
            put(getattr(t, into), int(t.table[0, at // 16]), at % 16, 5, x)
            got = t.run(hip, True)
            row = at - (lens[0] - chunk)  # the first row that sees it
            assert torch.isfinite(got[:row]).all()
            k, v = t.held()
            want, bound = ref.attention(t.q[:row].cpu(), k, v, t.table, [0, row], [at], d ** -0.5, True, P_UNIT[dtype])
            assert ((got[:row].cpu().double() - want).abs() <= ref.with_rounding(bound, want, DT[dtype])).all()
            if into == "v":
                assert torch.isfinite(got[..., :5]).all() and torch.isfinite(got[..., 6:]).all()
                seen = got[row:, :, 5]
                if x != x:
                    assert torch.isnan(seen).all()
                elif dtype == "bf16":
                    assert not torch.isfinite(seen).any()
                else:
                    assert (seen == x).all()
            elif x != x:
                assert torch.isnan(got[row:]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("chunk", [4, 90])
def test_nan_scores_stay_with_their_rows_from_the_first_key_on(hip, dtype, d, chunk):
    """A NaN in the first key makes every row of its head NaN, also those whose later tiles are clean, and no row of the
    other head; a NaN in a query makes that row NaN alone."""
    c = Case([chunk], [300], 2, 1, d, 16, dtype, False)
    clean = c.run(hip, True)
    c.q[chunk // 2, 0, 3] = float("nan")
    got = c.run(hip, True)
    assert torch.isnan(got[chunk // 2, 0]).all()
    got[chunk // 2, 0] = clean[chunk // 2, 0]
    assert torch.equal(got, clean)
    c.k[int(c.table[0, 0]), 1, 0, 0] = float("nan")
    got = c.run(hip, True)
    assert torch.isnan(got[:, 1]).all() and torch.equal(got[0, 0], clean[0, 0])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, 1.0, 0.02])
def test_scales_and_large_scores(hip, dtype, scale):
    c = Case([50], [200], 2, 2, 64, 16, dtype, False, spread=2.0)
    c.check(c.run(hip, True, scale=scale), True, scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_strided_queries_and_outputs(hip, dtype):
    c = Case([30, 4], [80, 20], 2, 2, 64, 16, dtype, False)
    want = c.run(hip, True)
    packed = torch.zeros(34, 3, 4, 64, device="cuda", dtype=DT[dtype])
    packed[:, 1] = c.q
    assert torch.equal(c.run(hip, True, q=packed[:, 1]), want)
    assert torch.equal(c.run(hip, True, q=c.q.transpose(1, 2).contiguous().transpose(1, 2)), want)
    off = torch.empty(c.q.numel() + 1, device="cuda", dtype=DT[dtype])[1:].view(c.q.shape).copy_(c.q)
    assert torch.equal(c.run(hip, True, q=off), want)
    out = torch.zeros(34, 3, 4, 64, device="cuda", dtype=DT[dtype])
    assert torch.equal(c.run(hip, True, out=out[:, 2]), want) and (out[:, :2] == 0).all()
    assert torch.equal(c.run(hip, True, out=c.q), want)  # in place


def test_shared_pages(hip):
    """Two sequences that share their first pages, and one page twice in a table, read alike."""
    c = Case([1, 1], [100, 100], 2, 2, 128, 16, "f16", False)
    c.table[1] = c.table[0]
    c.table[0, 3] = c.table[0, 2]
    c.table[1, 3] = c.table[0, 3]
    c.ti = c.table.cuda()
    c.q[1] = c.q[0]
    got = c.run(hip, True)
    assert torch.equal(got[0], got[1])
    c.check(got, True)


def test_refusals(hip):
    c = Case([4], [20], 2, 2, 64, 16, "f16", False)
    for call in (lambda: c.run(hip, True, q=c.q[:, :3]), lambda: c.run(hip, True, q=c.q.float()), lambda: c.run(hip, True, scale=-1.0),
                 lambda: c.run(hip, True, q=c.q[..., :32]), lambda: c.run(hip, True, out=c.q[:2]), lambda: c.run(hip, True, max_q=-1),
                 lambda: c.run(hip, True, scale=float("nan")), lambda: c.run(hip, True, q=c.q[0])):
        with pytest.raises(hip.SamHipError):
            call()
    assert c.run(hip, True, q=c.q[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_short_sequences_without_hints(hip, dtype):
    """A launch shaped by T and the table's width alone, whose workgroups mostly have nothing to do or several tiles."""
    chunks = [i * 7 % 9 for i in range(3000)]
    c = Case(chunks, [n + i * 5 % 8 for i, n in enumerate(chunks)], 4, 1, 64, 8, dtype, False)
    c.check(c.run(hip, True), True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [8, 16, 24, 40, 56, 88, 104, 120, 136, 248])
def test_many_rows_at_every_width_of_a_last_chunk(hip, dtype, d):
    """e4m3 rows in pieces of 16 codes, the last of them a half one, in the last row of the pool too."""
    c = Case([70, 40], [150, 64], 2, 1, d, 16, dtype, True, spare=0)
    for causal in (True, False):
        c.check(c.run(hip, causal), causal)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("chunks, lens, hkv, g, d", [
    ([300, 260, 7], [5000, 2600, 300], 1, 1, 64), ([600], [6000], 1, 2, 136), ([40], [2100], 1, 1, 256), ([3, 1], [9000, 600], 1, 2, 64)])
def test_more_than_eight_splits(hip, dtype, chunks, lens, hkv, g, d):
    """Key splits joined in a loop and by workgroups, with sequences that need fewer of them or one."""
    c = Case(chunks, lens, hkv, g, d, 16, dtype, False)
    hint = dict(max_q=max(chunks), max_len=max(lens))
    assert hip._paged_workspace(0, 1 if dtype == "f16" else 2, 1 if dtype == "f16" else 2, sum(chunks), len(chunks), hkv * g, hkv, d,
                                max(chunks), max(lens)) > 8 * sum(chunks) * hkv * g * d * 4
    for causal in (True, False):
        c.check(c.run(hip, causal, **hint), causal)


def test_sizes_past_32_bits_are_refused(hip):
    t = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt, device="cuda")
    i = lambda *s: t(*s, dt=torch.int32)
    big = 1 << 32
    kp = t(1, 1, 8, 8)
    with pytest.raises(hip.SamHipError, match="below 2\\^31"):
        hip.paged_attention(t(1, 1, 8), kp, kp, i(1, 1).expand(1, big), i(2), i(1))
    with pytest.raises(hip.SamHipError, match="below 2\\^31"):
        hip.paged_attention(t(1, 1, 8), kp, kp, i(1, 1), i(2), i(1), max_q=-1)
    with pytest.raises(hip.SamHipError, match="below 2\\^31"):
        hip.kv_read(kp, kp, i(1, 1), i(1), big)
    with pytest.raises(hip.SamHipError, match="below 2\\^31"):
        hip.kv_write(t(1, 1, 8).expand(big, 1, 8), t(1, 1, 8).expand(big, 1, 8), kp, kp.clone(), i(1, 1), i(2), i(1))
    with pytest.raises(hip.SamHipError, match="below 2\\^31"):
        hip.rope_axes(t(1, 1, 8).expand(big, 1, 8), i(1, 1), t(4, dt=torch.float64), i(4))
    assert hip.paged_attention(t(1, 1, 8), kp, kp, i(1, 1), torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                               torch.ones(1, dtype=torch.int32, device="cuda"), max_q=big, max_len=big).shape == (1, 1, 8)
