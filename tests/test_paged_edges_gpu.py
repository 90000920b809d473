"""The paged memory at the edges of what its header defines: weights far below a row's largest, scores of any size,
sequences that outgrow their table or the new tokens, results in place of their queries, e4m3 rows of every scale, empty
calls while the library is off."""
import math

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


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 20, 50])
@pytest.mark.parametrize("gap, length", [(16.0, 8192), (17.5, 8192), (17.5, 28736)])
def test_thousands_of_keys_far_below_a_dominant_one(hip, dtype, d, rows, gap, length):
    """A key of value 0 that holds nearly all of a row's weight, at either end, and thousands of equal ones `gap` nats
    lower, whose values are all that is left of the result. Scores are exact (0 and 8 * gap / 8), so that the bound is
    P's rounding in numerator and denominator, the sums' at one f32 rounding a key, an exponent's (4 roundings of
    gap log2 e), and the output's. (f16 weights of the many-row kernel leave the normal range at 2^-25 of the largest; at
    17.5 nats, 2^-25.25, half a subnormal step is 2^-10.75 of one, while the denominator, the dominant key, is exact.)"""
    dt, page = DT[dtype], 64
    w = math.exp(-gap)
    for first in (True, False):
        gen = torch.Generator(device="cuda").manual_seed(d + rows)
        k = torch.zeros(length, 1, d, device="cuda", dtype=dt)
        v = (0.5 + torch.rand(length, 1, d, generator=gen, device="cuda")).to(dt)
        at = 0 if first else length - 1
        k[at, 0, 0], v[at] = gap / 8, 0
        q = torch.zeros(rows, 1, d, device="cuda", dtype=dt)
        q[:, 0, 0] = 8
        pages = -(-length // page)
        kp, vp = (torch.zeros(pages, 1, page, d, device="cuda", dtype=dt) for _ in range(2))
        table = torch.arange(pages, device="cuda", dtype=torch.int32).view(1, -1)
        hip.kv_write(k, v, kp, vp, table, ints([0, length]), ints([length]))
        got = hip.paged_attention(q, kp, vp, table, ints([0, rows]), ints([length]), scale=1.0, causal=False)
        want = (v.double().sum(0) * w / (1 + (length - 1) * w)).expand(rows, 1, d).cpu()
        rel = 2 * P_UNIT[dtype] + (length + 16) * ref.F32_U + 2 * 4 * gap * ref.F32_U
        bound = ref.with_rounding(rel * want, want, dt)
        assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 20, 50])
@pytest.mark.parametrize("power, scale", [(19, 1.0), (21, 0.37), (24, 0.37), (28, 1.0), (30, 1.0), (30, 0.37)])
def test_scores_of_any_size(hip, dtype, d, rows, power, scale):
    """Scores of 0 and +- 2^power, exact in f32: the largest ones share all the weight evenly (the others are 2^18 nats lower
    at least), wherever they lie and whether the maximum is reached from below, at once or is a negative one. The bound
    is P's rounding, the sums' at one f32 rounding a key and the output's."""
    dt, page, length = DT[dtype], 16, 3000
    gen = torch.Generator(device="cuda").manual_seed(d + rows)
    v = torch.randn(length, 1, d, generator=gen, device="cuda").to(dt)
    q = torch.zeros(rows, 1, d, device="cuda", dtype=dt)
    q[:, 0, 0] = 2.0 ** (power // 2)
    pages = -(-length // page)
    kp, vp = (torch.zeros(pages, 1, page, d, device="cuda", dtype=dt) for _ in range(2))
    table = torch.arange(pages, device="cuda", dtype=torch.int32).view(1, -1)
    at = torch.arange(length, device="cuda")
    pair = (at == 5) | (at == 2950)
    for step in (torch.where(pair, 1, -1), torch.where(pair, -1, 1), torch.where(at < 300, -1, 0), torch.where(at < 300, 0, 1),
                 torch.where(pair, 0, -1), torch.full_like(at, -1)):
        k = torch.zeros(length, 1, d, device="cuda", dtype=dt)
        k[:, 0, 0] = step * 2.0 ** (power - power // 2)
        hip.kv_write(k, v, kp, vp, table, ints([0, length]), ints([length]))
        got = hip.paged_attention(q, kp, vp, table, ints([0, rows]), ints([length]), scale=scale, causal=False).cpu().double()
        top = v[step == step.max()].double()
        want, spread = (x.mean(0).expand(rows, 1, d).cpu() for x in (top, top.abs()))
        bound = ref.with_rounding((2 * P_UNIT[dtype] + (length + 16) * ref.F32_U) * spread, want, dt)
        assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 50])
def test_scores_of_any_size_from_e4m3_pages(hip, dtype, d, rows):
    """As above from 8 bits (scores of 2^30 are powers of two there too), the values as they are read back."""
    dt, page, length = DT[dtype], 16, 3000
    gen = torch.Generator(device="cuda").manual_seed(d + rows)
    v = torch.randn(length, 1, d, generator=gen, device="cuda").to(dt)
    q = torch.zeros(rows, 1, d, device="cuda", dtype=dt)
    q[:, 0, 0] = 2.0 ** 15
    pages = -(-length // page)
    kp, vp = (torch.zeros(pages, 1, page, d, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((pages, 1, page), 127, device="cuda", dtype=torch.uint8) for _ in range(2))
    table = torch.arange(pages, device="cuda", dtype=torch.int32).view(1, -1)
    at = torch.arange(length, device="cuda")
    pair = (at == 5) | (at == 2950)
    for step in (torch.where(pair, 1, -1), torch.where(pair, -1, 1), torch.where(at < 300, -1, 0)):
        k = torch.zeros(length, 1, d, device="cuda", dtype=dt)
        k[:, 0, 0] = step * 2.0 ** 15
        hip.kv_write(k, v, kp, vp, table, ints([0, length]), ints([length]), ks, vs)
        held = hip.kv_read(kp, vp, table, ints([length]), length, ks, vs, dtype=dt)[1][0]
        got = hip.paged_attention(q, kp, vp, table, ints([0, rows]), ints([length]), ks, vs, scale=1.0, causal=False).cpu().double()
        top = held[step == step.max()].double()
        want, spread = (x.mean(0).expand(rows, 1, d).cpu() for x in (top, top.abs()))
        bound = ref.with_rounding((2 * P_UNIT[dtype] + (length + 16) * ref.F32_U) * spread, want, dt)
        assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("chunk", [1, 20, 150])
def test_scores_of_any_size_keep_masks_and_values_apart(hip, dtype, d, chunk):
    """Scores that grow by 2^22 a key: a causal row is its own key's value, and a NaN at one position reaches the rows from
    there on, in its column alone."""
    dt, page, length, col, bad = DT[dtype], 16, 190, 3, 187
    gen = torch.Generator(device="cuda").manual_seed(d + chunk)
    v = torch.randn(length, 1, d, generator=gen, device="cuda").to(dt)
    v[bad, 0, col] = float("nan")
    k = torch.zeros(length, 1, d, device="cuda", dtype=dt)
    k[:, 0, 0] = torch.arange(length, device="cuda") * 2.0 ** 8
    q = torch.zeros(chunk, 1, d, device="cuda", dtype=dt)
    q[:, 0, 0] = 2.0 ** 14
    kp, vp = (torch.full((12, 1, page, d), float("nan"), device="cuda", dtype=dt) for _ in range(2))
    table = torch.arange(12, device="cuda", dtype=torch.int32).view(1, -1)
    hip.kv_write(k, v, kp, vp, table, ints([0, length]), ints([length]))
    got = hip.paged_attention(q, kp, vp, table, ints([0, chunk]), ints([length]), scale=1.0).cpu().double()
    at = torch.arange(length - chunk, length)
    want = v[length - chunk:].cpu().double()
    assert torch.equal(torch.isnan(got[:, 0, col]), at >= bad)
    got[at >= bad, 0, col], want[at >= bad, 0, col] = 0, 0
    bound = ref.with_rounding((2 * P_UNIT[dtype] + (length + 16) * ref.F32_U) * want.abs(), want, dt)
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [1, 4, 40])
def test_a_sequence_that_outgrows_its_table_or_its_tokens(hip, dtype, heads):
    """kv_write and paged_attention give a token one position: lens past what the table names, and starts past the
    tokens (whose last ones are not there), move no token that fits. lens 70 over a table of 64: tokens 0 .. 13 of 20
    are stored at 50 .. 63, token t sees keys to 50 + t, those behind the table's end all 64."""
    dt, d, page = DT[dtype], 64, 16
    gen = torch.Generator(device="cuda").manual_seed(heads)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dt)
    for chunk, end, length in ((20, 20, 70), (20, 26, 60), (20, 26, 68), (12, 12, 70), (20, 20, 2 ** 31 - 1), (20, 2 ** 31 - 1, 5),
                               (20, 2 ** 31 - 1, -2 ** 31)):
        kp, vp = rnd(4, 1, page, d), rnd(4, 1, page, d)
        table = ints([[2, 0, 3, 1]])
        q, k, v = rnd(chunk, heads, d), rnd(chunk, 1, d), rnd(chunk, 1, d)
        hip.kv_write(k, v, kp, vp, table, ints([0, end]), ints([length]))
        got = hip.paged_attention(q, kp, vp, table, ints([0, end]), ints([length])).cpu().double()
        for t in range(chunk):
            at = length - end + t  # its position
            if 0 <= at < 64:
                assert torch.equal(kp[int(table[0, at // page]), 0, at % page], k[t, 0])
            want, bound = ref.attention(q[t:t + 1].cpu(), kp.cpu(), vp.cpu(), table.cpu(), [0, 1], [min(at + 1, 64)],
                                        d ** -0.5, True, P_UNIT[dtype])
            assert ((got[t:t + 1] - want).abs() <= ref.with_rounding(bound, want, dt)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("chunks, lens, d", [([1, 1], [3000, 40], 128), ([300, 70], [300, 2000], 64), ([20, 5], [4000, 9], 256)])
def test_results_in_place_of_their_queries(hip, dtype, chunks, lens, d):
    """out = q, contiguous and as a part of packed rows, with split keys and without, equals a result apart bit for bit; the
    rest of the packed rows stays."""
    dt, page, t = DT[dtype], 16, sum(chunks)
    gen = torch.Generator(device="cuda").manual_seed(d)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dt)
    width = -(-max(lens) // page)
    kp, vp = rnd(2 * width, 2, page, d), rnd(2 * width, 2, page, d)
    args = kp, vp, torch.arange(2 * width, device="cuda", dtype=torch.int32).view(2, -1), ints([0, chunks[0], t]), ints(lens)
    packed = rnd(t, 3, 4, d)
    q = packed[:, 1].contiguous()
    for causal in (True, False):
        want = hip.paged_attention(q, *args, causal=causal)
        own, rows = q.clone(), packed.clone()
        assert hip.paged_attention(own, *args, causal=causal, out=own) is own and torch.equal(own, want)
        hip.paged_attention(rows[:, 1], *args, causal=causal, out=rows[:, 1])
        assert torch.equal(rows[:, 1], want) and torch.equal(rows[:, ::2], packed[:, ::2])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_an_e4m3_row_is_read_as_kv_read_returns_it(hip, dtype, d, rows):
    """With one visible key the attention is that key's value, in q's dtype as kv_read rounds it: for each scale that
    kv_write makes (bytes 1 .. 253), codes of every size, results past the type's range and below its normal one."""
    dt, b = DT[dtype], 253
    gen = torch.Generator(device="cuda").manual_seed(d)
    codes = torch.randint(0, 256, (b, 1, 1, d), generator=gen, device="cuda", dtype=torch.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x7E  # the largest value in place of NaN
    v = codes.view(torch.float8_e4m3fn)
    k = torch.zeros(b, 1, 1, d, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    vs = torch.arange(1, b + 1, device="cuda", dtype=torch.int32).to(torch.uint8).view(b, 1, 1)
    ks = torch.full((b, 1, 1), 127, device="cuda", dtype=torch.uint8)
    table, lens = torch.arange(b, device="cuda", dtype=torch.int32).view(b, 1), ints([1] * b)
    _, want = hip.kv_read(k, v, table, lens, 1, ks, vs, dtype=dt)
    q = torch.randn(b * rows, 1, d, generator=gen, device="cuda").to(dt)
    starts = torch.arange(b + 1, device="cuda", dtype=torch.int32) * rows
    got = hip.paged_attention(q, k, v, table, starts, lens, ks, vs, causal=False, max_q=rows)
    got, want = got.view(b, rows, d), want.view(b, 1, d).expand(b, rows, d)
    bad = (got != want).any(-1).any(-1).nonzero().flatten().tolist()
    assert not bad, f"scale bytes {[x + 1 for x in bad]}"


def test_calls_without_work_obey_the_switch(hip):
    """No tokens, no sequences, no pages in the table, no columns to read: while the library is off each call raises, and
    otherwise returns its empty or zero result."""
    h = lambda *s: torch.ones(s, device="cuda", dtype=torch.float16)
    pages, x, table = h(3, 2, 16, 64), h(4, 2, 64), ints([[0, 1]])
    s, n, none = ints([0, 4]), ints([4]), (ints([]).view(0, 2), ints([0]), ints([]))
    freqs, axes = hip.rope_freqs((8, 8))
    calls = [lambda: hip.rope_axes(x[:0], ints([]).view(0, 2), freqs, axes), lambda: hip.kv_write(x[:0], x[:0], pages, pages, table, s, n),
             lambda: hip.kv_write(x, x, pages, pages, *none), lambda: hip.kv_write(x, x, pages, pages, table[:, :0], s, n),
             lambda: hip.kv_read(pages, pages, table, n, 0)[0], lambda: hip.kv_read(pages, pages, table[:, :0], n, 4)[0],
             lambda: hip.kv_read(pages, pages, none[0], none[2], 4)[0], lambda: hip.paged_attention(x[:0], pages, pages, table, s, n),
             lambda: hip.paged_attention(x, pages, pages, *none), lambda: hip.paged_attention(x, pages, pages, table[:, :0], s, n)]
    shapes = [(0, 2, 64), None, None, None, (1, 0, 2, 64), (1, 4, 2, 64), (0, 4, 2, 64), (0, 2, 64), (4, 2, 64), (4, 2, 64)]
    hip.set_enabled(False)
    try:
        for call in calls:
            with pytest.raises(hip.SamHipDisabled, match="switched off"):
                call()
    finally:
        hip.set_enabled(True)
    for call, shape in zip(calls, shapes):
        got = call()
        assert got is None if shape is None else got.shape == shape and not got.any()
