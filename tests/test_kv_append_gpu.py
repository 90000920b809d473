"""kv_append on an MI355X: queries within the turn's bound, keys rounded once from the turn in 64 bits (codes and scales are
the definition's), values as kv_write stores them, everything else untouched."""
import pytest
import torch

import mx_ref
import paged_ref as ref
from test_e2m1_cache_gpu import E2M1
from test_e2m1_cache_gpu import pool as pool4
from test_kv_cache_gpu import pool, tables

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


def a_pool(held, pages, heads, page, d, dt):
    return pool4(pages, heads, page, d, 3, (0, 255)) if held == "e2m1" else pool(pages, heads, page, d, dt, held == "e4m3")


def as_held(x, held, dt):
    """(bytes that a pool holds for rows of x in 64 bits, scale bytes)."""
    if held == "e2m1":
        _, codes, exps = mx_ref.quantise(x)
        return mx_ref.packed(codes), exps
    if held == "e4m3":
        val, exps = ref.quantise(x)
        two = torch.pow(torch.tensor(2.0, dtype=torch.float64), exps.double() - 127)[..., None]
        return (val / two).float().to(torch.float8_e4m3fn).view(torch.uint8), exps  # exact: val / two is an e4m3 value
    return (x.to(dt) if dt != torch.float32 else x.float()), None


def one_rounding(x, dt):
    """x (64 bits) rounded to dt once: through f32 rounded to odd."""
    f = x.float()
    bits = f.view(torch.int32)
    away = f.double().abs() > x.abs()
    odd = torch.where(f.double() == x, bits, (bits - away.int()) | 1).view(torch.float32)
    return f if dt == torch.float32 else odd.to(dt)


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


CASES = [  # chunks, lens, query heads, key heads, d, page, turned pairs, axes (0: the tokens' own positions)
    ([1], [1], 1, 1, 64, 16, 32, 0), ([5, 0, 3], [5, 7, 40], 6, 3, 96, 8, 48, 3), ([130], [577], 8, 2, 128, 24, 64, 0),
    ([1] * 70, list(range(1, 71)), 2, 2, 64, 16, 16, 1), ([40, 9], [40, 100], 1, 1, 256, 100, 128, 2), ([3, 3, 3], [3, 5, 64], 5, 5, 32, 1, 13, 2),
    ([64, 1], [64, 65], 12, 4, 160, 64, 61, 6), ([7], [7], 7, 7, 224, 256, 0, 1), ([2500, 30], [2600, 5000], 16, 4, 128, 16, 64, 0),
    ([1], [30], 32, 8, 128, 16, 1, 3), ([900], [900], 10, 5, 64, 32, 20, 4)]


def inputs(case, dtype, pairs, seed=1):
    chunks, lens, hq, hkv, d, page, turned, naxes = case
    dt, t = DT[dtype], sum(chunks)
    g = torch.Generator(device="cuda").manual_seed(seed + d + t)
    rnd = lambda h: torch.randn(t, h, d, generator=g, device="cuda")
    k = (rnd(hkv) * torch.pow(10.0, torch.randint(-2, 3, (t, hkv, 1), generator=g, device="cuda").float())).to(dt)
    freqs = torch.tensor([10000.0 ** (-i / max(1, turned)) for i in range(turned)], dtype=torch.float64, device="cuda")
    axes = torch.randint(-1, max(1, naxes) + 1, (turned,), generator=g, device="cuda").int() if naxes else torch.zeros(turned, device="cuda").int()
    pos = torch.randint(-(1 << 20), 1 << 20, (t, naxes), generator=g, device="cuda").int() if naxes else None
    if pos is not None:
        pos[0] = 0
    return rnd(hq).to(dt), k, rnd(hkv).to(dt), freqs, axes, pos


def turned_64(x, freqs, axes, pos, at, pairs):
    x, out = x.cpu().double(), x.cpu().double().clone()
    p = len(freqs)
    for i in range(p):
        ax = int(axes[i])
        where = at if pos is None else pos.cpu()[:, ax] if 0 <= ax < pos.shape[1] else torch.zeros(len(x))
        a = (where.double() * float(freqs[i]))[:, None]
        lo, hi = (2 * i, 2 * i + 1) if pairs == "adjacent" else (i, i + p)
        out[..., lo] = x[..., lo] * a.cos() - x[..., hi] * a.sin()
        out[..., hi] = x[..., hi] * a.cos() + x[..., lo] * a.sin()
    return out


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("case", CASES)
def test_matches_the_definition(hip, held, dtype, pairs, case):
    chunks, lens, hq, hkv, d, page, turned, naxes = case
    dt = DT[dtype]
    q, k, v, freqs, axes, pos = inputs(case, dtype, pairs)
    width = -(-max(lens) // page) + 1
    pages = sum(-(-n // page) for n in lens) + 4
    table, starts = tables(chunks, lens, page, width, pages)
    kp, vp, ks, vs = a_pool(held, pages, hkv, page, d, dt)
    before = [x.clone() for x in (kp, vp, ks, vs) if x is not None]
    ti, si, li = table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    got = hip.kv_append(q, k, v, freqs, axes, kp, vp, ti, si, li, ks, vs, pos, pairs)
    places = [(b, at) for b in range(len(lens)) for at in ref.positions(starts, lens, b)]
    at = torch.tensor([a for _, a in places])
    # queries: sine and cosine are f32 roundings of exact ones, the turn rounds twice more in f32 (paged_ref.rope_bound allows
    # its own, wider, error of both)
    want = turned_64(q, freqs, axes, pos, at, pairs)
    bound = ref.rope_bound(q.cpu(), want, turned, pairs, dt)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert torch.equal(got[..., 2 * turned:], q[..., 2 * turned:])
    # keys: the 64-bit turn rounded once. The kernel's 64-bit turn differs from this one in its last bits, so a value within
    # 2^-44 of a border between two roundings may go either way: none of some hundred thousand does (chance below 1e-7)
    page_of = torch.tensor([int(table[b, a // page]) for b, a in places])
    slot = torch.tensor([a % page for _, a in places])
    new = turned_64(k, freqs, axes, pos, at, pairs)
    touched = torch.zeros(pages, page, dtype=torch.bool)
    touched[page_of, slot] = True
    for x, p, s in ((new, kp, ks), (v.cpu().double(), vp, vs)):
        codes, exps = as_held(x, held, dt) if held != "own" else (one_rounding(x, dt), None)
        raw = p.cpu() if held == "own" else p.cpu().view(torch.uint8)
        assert same_bytes(raw[page_of, :, slot], codes) or torch.equal(raw[page_of, :, slot].double(), codes.double())
        if exps is not None:
            assert torch.equal(s.cpu()[page_of, :, slot], exps)
    for x, old in zip([x for x in (kp, vp, ks, vs) if x is not None], before):
        a, o = x.cpu().view(torch.uint8).transpose(1, 2), old.cpu().view(torch.uint8).transpose(1, 2)
        assert torch.equal(a[~touched], o[~touched])


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_position_zero_stores_what_kv_write_stores(hip, held, dtype):
    """No turn: the same bytes as kv_write, for ties, extremes and values that are not finite."""
    dt = DT[dtype]
    f = torch.finfo(dt)
    rows = [torch.linspace(-448, 448, 64), torch.linspace(-6, 6, 64), torch.full((64,), f.max), torch.full((64,), f.tiny), torch.zeros(64),
            torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 8), torch.full((64,), f.smallest_normal * f.eps),
            torch.tensor([450.0] + [1e-3] * 63), torch.tensor([17.0, 19.0, 448.0, 432.0] * 16)]
    x = torch.stack(rows).to(dt).cuda().view(-1, 1, 64)
    bad = x.clone()
    bad[1, 0, 5], bad[3, 0, 40], bad[4, 0, 63] = float("nan"), float("inf"), -float("inf")
    n = len(rows)
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    freqs, axes = hip.rope_freqs((32,))
    for turned, k in ((freqs, x), (freqs[:0], x), (freqs[:0], bad)):
        for pairs in ("adjacent", "halves"):
            a, b = a_pool(held, 1, 1, n, 64, dt), a_pool(held, 1, 1, n, 64, dt)
            q = hip.kv_append(k, k, bad, turned, axes[:len(turned)], a[0], a[1], i(0).view(1, 1), i(0, n), i(n), a[2], a[3], torch.zeros(1, 1, device="cuda").int(), pairs)
            hip.kv_write(k, bad, b[0], b[1], i(0).view(1, 1), i(0, n), i(n), b[2], b[3])
            assert same_bytes(q, k)
            for u, w in zip(a, b):
                assert u is None or same_bytes(u, w)


def test_values_that_are_not_finite_in_keys(hip):
    """A NaN or an infinity in a turned pair reaches both of its columns, and no others."""
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    freqs, axes = hip.rope_freqs((16,))
    for pairs, partner in (("adjacent", 7), ("halves", 22)):
        x = torch.randn(3, 2, 64, device="cuda").half()
        x[1, 1, 6] = float("nan")
        x[2, 0, 40] = float("inf")  # not turned
        kp, vp, _, _ = pool(1, 2, 8, 64, torch.float16, False)
        q = hip.kv_append(x, x, x, freqs, axes, kp, vp, i(0).view(1, 1), i(0, 3), i(8), pairs=pairs)
        for y in (q, kp[0, :, 5:8].transpose(0, 1)):
            off = torch.zeros(3, 2, 64, dtype=torch.bool, device="cuda")
            off[1, 1, 6], off[1, 1, partner], off[2, 0, 40] = True, True, True
            assert torch.equal(~torch.isfinite(y), off)


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
def test_strides_views_in_place_and_no_queries(hip, held):
    case = ([30, 4], [80, 20], 4, 2, 64, 16, 24, 0)
    q, k, v, freqs, axes, _ = inputs(case, "f16", "halves")
    table, starts = tables(case[0], case[1], 16, 5, 12)
    ti, si, li = table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(case[1], dtype=torch.int32).cuda()
    for pairs in ("adjacent", "halves"):
        def call(q, k, v, **kw):
            p = a_pool(held, 12, 2, 16, 64, torch.float16)
            return hip.kv_append(q, k, v, freqs, axes, p[0], p[1], ti, si, li, p[2], p[3], pairs=pairs, **kw), p

        want, pages = call(q, k, v)
        packed = torch.cat([q, k, v], 1)  # one projection's output
        for got, p in (call(packed[:, :4], packed[:, 4:6], packed[:, 6:]),
                       call(q.transpose(1, 2).contiguous().transpose(1, 2), torch.empty(k.numel() + 1, device="cuda", dtype=torch.float16)[1:].view(k.shape).copy_(k), v),
                       call(q.clone(), k, v, out=torch.zeros(34, 3, 4, 64, device="cuda", dtype=torch.float16)[:, 1])):
            assert torch.equal(got, want) and all(u is None or same_bytes(u, w) for u, w in zip(p, pages))
        for inplace in (q.clone(), packed.clone()[:, :4]):
            got, p = call(inplace, k, v, out=inplace)
            assert got is inplace and torch.equal(got, want)
        none, p = call(None, k, v)
        assert none is None and all(u is None or same_bytes(u, w) for u, w in zip(p, pages))
        # positions that broadcast
        pos = torch.full((1, 1), 5, device="cuda", dtype=torch.int32)
        assert torch.equal(call(q, k, v, pos=pos)[0], call(q, k, v, pos=pos.expand(34, 1).contiguous())[0])


def test_tokens_outside_and_places_that_are_not_there(hip):
    q, k = torch.ones(12, 2, 64, device="cuda", dtype=torch.float16), torch.ones(12, 1, 64, device="cuda", dtype=torch.float16)
    freqs, axes = hip.rope_freqs((32,))
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    kp, vp, _, _ = pool(3, 1, 4, 64, torch.float16, False)
    old = kp.clone()
    run = lambda t, s, n, **kw: hip.kv_append(q, k, k, freqs, axes, kp, vp, i(t), i(s), i(n), **kw)
    a = run([[7, -1], [3, 1 << 30]], [0, 4, 8], [8, 8])
    assert (a[8:] == 0).all() and not (a[:8] == 0).all()
    for t, s, n in (([[0, 1], [2, -5]], [0, 4, 8], [-3, 0]), ([[0, 1], [2, -5]], [0, 4, 8], [1 << 30, 2 ** 31 - 1]), ([[0, 1]], [12, 12], [4]),
                    ([[0, 1]], [-7, 0], [4])):
        run(t, s, n)
    assert torch.equal(kp, old)
    kept = torch.full_like(q, 3.0)
    run([[0, 1], [2, -5]], [2, 4, 10], [1, 6], out=kept)  # one of 2 fits; 4 of 6 have a page
    assert (kept[:2] == 3).all() and (kept[10:] == 3).all() and not (kept[2:10] == 3).any()
    got = kp[:, 0, :, 0] != old[:, 0, :, 0]
    assert got.tolist() == [[True, False, False, False], [False] * 4, [True] * 4]
    # a token before its sequence's start has its query turned by that negative position
    want = hip.rope_axes(q[2:3], i([[-1]]), freqs, axes)
    assert torch.allclose(kept[2:3], want, atol=2e-3)
    assert hip.kv_append(q[:0], k[:0], k[:0], freqs, axes, kp, vp, i([[0]]), i([0, 0]), i([4])).shape == (0, 2, 64)
    assert (hip.kv_append(q, k, k, freqs, axes, kp, vp, i([[0]])[:0], i([0]), i([])) == 0).all()
    assert torch.equal(hip.kv_append(q, k, k, freqs, axes, kp, vp, i([[0]])[:, :0], i([0, 12]), i([12])),
                       hip.rope_axes(q, torch.arange(12, device="cuda").int()[:, None], freqs, axes))


def test_far_positions_keep_their_angles(hip):
    """Positions up to 2^31 and frequencies above 1: the key is the 64-bit turn of the f64 product, to half a step."""
    t = 300
    g = torch.Generator(device="cuda").manual_seed(0)
    k = torch.randn(t, 1, 64, generator=g, device="cuda")
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (t, 1), generator=g, device="cuda").int()
    freqs, axes = hip.rope_freqs((32,), scale=3.0)
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    kp, vp, _, _ = pool(1, 1, t, 64, torch.float32, False)
    hip.kv_append(None, k, k, freqs, axes, kp, vp, i(0).view(1, 1), i(0, t), i(t), pos=pos)
    want = turned_64(k, freqs, axes, pos, None, "adjacent")[:, 0]
    # an angle of 2^33 in f64 is exact as a number; sine and cosine to 2^-50, so f32's half step and a little
    assert ((kp[0, 0].cpu().double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -46).all()


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
def test_pages_past_4_gib(hip, held):
    """The last pages of pools of more than 2^32 bytes hold what the first ones do, and their neighbours stay."""
    pages, heads, page, d, n = 72000, 8, 128, 128, 200
    dt = {"own": torch.float16, "e4m3": torch.float8_e4m3fn, "e2m1": E2M1}[held]
    raw = [torch.zeros(pages, heads, page, d * 2 if held == "own" else d if held == "e4m3" else d // 2, device="cuda", dtype=torch.uint8) for _ in range(2)]
    kp, vp = (x.view(dt) for x in raw)
    scales = [None, None] if held == "own" else [torch.zeros(pages, heads, page, *((d // 32,) if held == "e2m1" else ()), device="cuda", dtype=torch.uint8) for _ in range(2)]
    assert raw[0].numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda").half() for h in (16, heads, heads))
    freqs, axes = hip.rope_freqs((64,))
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    got = [hip.kv_append(q, k, v, freqs, axes, kp, vp, table.view(1, 2), i(0, n), i(n), *scales) for table in (i(pages - 1, pages - 2), i(0, 1))]
    assert torch.equal(*got)
    for x in raw + [s for s in scales if s is not None]:
        assert torch.equal(x[-1], x[0]) and torch.equal(x[-2], x[1]) and x[0].any() and not x[2].any() and not x[-3].any()


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
def test_a_decoding_loop_in_a_graph(hip, held):
    """kv_append and paged_attention as a decoder calls them, captured once and replayed as its lengths grow, against the
    eager calls; and a step's results against the whole sequence's in one call."""
    hq, hkv, d, page, n = 8, 2, 64, 16, 40
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda h: torch.randn(2, n, h, d, generator=g, device="cuda").bfloat16()
    q, k, v = rnd(hq), rnd(hkv), rnd(hkv)
    freqs, axes = hip.rope_freqs((32,))
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = i([[0, 2, 4], [1, 3, 5]])
    whole, one, again = (a_pool(held, 6, hkv, page, d, torch.bfloat16) for _ in range(3))
    for p in (whole, one, again):
        for x in p:
            if x is not None:
                x.view(torch.uint8).zero_()

    def step(p, q, k, v, starts, lens, max_q):
        qr = hip.kv_append(q, k, v, freqs, axes, p[0], p[1], table, starts, lens, p[2], p[3], pairs="halves")
        return hip.paged_attention(qr, p[0], p[1], table, starts, lens, p[2], p[3], max_q=max_q, max_len=n)

    flat = lambda x: x.reshape(2 * n, *x.shape[2:])
    all_at_once = step(whole, flat(q), flat(k), flat(v), i([0, n, 2 * n]), i([n, n]), n).view(2, n, hq, d)
    sq, sk, sv, lens, starts = q[:, 0].clone(), k[:, 0].clone(), v[:, 0].clone(), i([1, 1]), i([0, 1, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(one, sq, sk, sv, starts, lens, 1)
    for j in range(n):
        sq.copy_(q[:, j]), sk.copy_(k[:, j]), sv.copy_(v[:, j])
        lens.fill_(j + 1)
        graph.replay()
        eager = step(again, q[:, j], k[:, j], v[:, j], starts, i([j + 1, j + 1]), 1)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        # the same keys and values, in sums of another order: bf16's rounding of the result and P's two terms
        assert torch.allclose(out.float(), all_at_once[:, j].float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    for a, b, c in zip(whole, one, again):
        assert a is None or (same_bytes(a, b) and same_bytes(a, c))


def test_two_streams_and_repeats(hip):
    case = CASES[8]
    calls = []
    for dtype, held, seed in (("f16", "e2m1", 1), ("bf16", "e4m3", 9)):
        q, k, v, freqs, axes, _ = inputs(case, dtype, "halves", seed)
        table, starts = tables(case[0], case[1], 16, 320, 700)
        p = a_pool(held, 700, 4, 16, 128, DT[dtype])
        calls.append((q, k, v, freqs, axes, p[0], p[1], table.cuda(), torch.tensor(starts).int().cuda(), torch.tensor(case[1]).int().cuda(), p[2], p[3], None, "halves"))
    want = [(hip.kv_append(*c).clone(), *(c[n].view(torch.uint8).clone() for n in (5, 6, 10, 11))) for c in calls]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, c in zip(side, calls):
            with torch.cuda.stream(s):
                got.append(hip.kv_append(*c))
        torch.cuda.synchronize()
        for y, c, w in zip(got, calls, want):
            assert torch.equal(y, w[0]) and all(torch.equal(c[n].view(torch.uint8), x) for n, x in zip((5, 6, 10, 11), w[1:]))


def test_refusals(hip):
    q, k = torch.zeros(2, 4, 64, device="cuda", dtype=torch.float16), torch.zeros(2, 1, 64, device="cuda", dtype=torch.float16)
    kp, vp, _, _ = pool(3, 1, 4, 64, torch.float16, False)
    freqs, axes = hip.rope_freqs((32,))
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    t, s, n = i([[0, 1]]), i([0, 2]), i([2])
    ok = dict(q=q, k=k, v=k, freqs=freqs, axes=axes, k_pages=kp, v_pages=vp, table=t, starts=s, lens=n)
    for change in ({"q": q.float()}, {"q": q[:1]}, {"q": q[..., :32]}, {"q": q[:, :0]}, {"k": k[:1]}, {"k": k.float()}, {"v": k.bfloat16()}, {"freqs": freqs.float()},
                   {"axes": axes.long()}, {"axes": axes[:3]}, {"freqs": torch.zeros(33, dtype=torch.float64, device="cuda"), "axes": torch.zeros(33, device="cuda").int()},
                   {"pos": i([[1, 2, 3]]).float()}, {"pos": i([[1], [2], [3]])}, {"pos": i([[], []])}, {"pairs": "rows"}, {"out": q[:1]}, {"out": q.float()},
                   {"q": None, "out": q}, {"starts": s[:1]}, {"lens": n.long()}, {"table": t.cpu()}, {"k_scale": kp}, {"out": q[:, :1].expand(2, 4, 64)},
                   {"out": q.transpose(1, 2).contiguous().transpose(1, 2)}):
        with pytest.raises(hip.SamHipError):
            hip.kv_append(**{**ok, **change})
    with pytest.raises(hip.SamHipError, match="key heads"):
        hip.kv_append(**{**ok, "k": k[:, :0], "v": k[:, :0], "k_pages": kp[:, :0], "v_pages": vp[:, :0]})
    hip.set_enabled(False)
    try:
        for change in ({}, {"q": q[:0], "k": k[:0], "v": k[:0]}):
            with pytest.raises(hip.SamHipDisabled):
                hip.kv_append(**{**ok, **change})
    finally:
        hip.set_enabled(True)
