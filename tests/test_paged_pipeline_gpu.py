"""The paged memory as a program uses it, on an MI355X: a video's frames and objects of different ages written, turned and
attended step by step; captured graphs; streams; calls that repeat their bits."""
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


class Memory:
    """A paged cache of `heads` key heads for `batch` sequences and the steps that a program takes with it."""

    def __init__(self, hip, batch, heads, group, d, page, width, dtype, fp8, device="cuda"):
        self.hip, self.heads, self.group, self.d = hip, heads, group, d
        pages = batch * width
        kind = torch.float8_e4m3fn if fp8 else dtype
        self.k, self.v = (torch.zeros(pages, heads, page, d, device=device, dtype=torch.uint8 if fp8 else kind) for _ in range(2))
        self.ks = self.vs = None
        if fp8:
            self.k, self.v = self.k.view(kind), self.v.view(kind)
            self.ks, self.vs = (torch.full((pages, heads, page), 127, device=device, dtype=torch.uint8) for _ in range(2))
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(9)).to(torch.int32).view(batch, width).to(device)
        self.freqs, self.axes = hip.rope_freqs((d // 8, d // 8, d // 4), device=device)

    def step(self, q, k, v, pos, starts, lens, causal=True, **kw):
        """Turns the new queries and keys, stores keys and values, attends."""
        q, k = self.hip.rope_axes(q, pos, self.freqs, self.axes), self.hip.rope_axes(k, pos, self.freqs, self.axes)
        self.hip.kv_write(k, v, self.k, self.v, self.table, starts, lens, self.ks, self.vs)
        return self.hip.paged_attention(q, self.k, self.v, self.table, starts, lens, self.ks, self.vs, causal=causal, **kw)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fp8", [False, True])
def test_steps_equal_the_formula_on_everything_written(hip, dtype, fp8):
    """Three steps (a prompt, a token each, a chunk each) of three sequences; after each, the attention equals the
    definition on the turned keys and values as they were stored, which are kept beside the cache and never read from it."""
    dt, heads, group, d, page = DT[dtype], 2, 3, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(0)
    m = Memory(hip, 3, heads, group, d, page, 16, dt, fp8)
    kept = [([], []) for _ in range(3)]
    lens = [0, 0, 0]
    for chunks in ([70, 5, 33], [1, 1, 1], [20, 64, 3]):
        t = sum(chunks)
        q, k, v = randn(gen, dt, t, heads * group, d), randn(gen, dt, t, heads, d), randn(gen, dt, t, heads, d)
        pos = torch.randint(0, 100, (t, 3), generator=gen, device="cuda", dtype=torch.int32)
        starts = [sum(chunks[:i]) for i in range(4)]
        lens = [n + c for n, c in zip(lens, chunks)]
        got = m.step(q, k, v, pos, ints(*starts), ints(*lens))
        qt, kt = (hip.rope_axes(x, pos, m.freqs, m.axes).cpu() for x in (q, k))
        for b in range(3):
            for i, x in enumerate((kt, v.cpu())):
                rows = x[starts[b]:starts[b + 1]]
                kept[b][i].append(ref.quantise(rows)[0].to(dt) if fp8 else rows)
        p_unit = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -16}[dtype]
        for b in range(3):
            k1, v1 = (torch.cat(x).transpose(0, 1)[None] for x in kept[b])  # one page that holds the sequence
            want, bound = ref.attention(qt[starts[b]:starts[b + 1]], k1, v1, torch.zeros(1, 1, dtype=torch.int32),
                                        [0, chunks[b]], [lens[b]], d ** -0.5, True, p_unit)
            off = (got[starts[b]:starts[b + 1]].cpu().double() - want).abs()
            assert (off <= ref.with_rounding(bound, want, dt)).all()


def test_a_ring_of_frames_is_the_memory_attention(hip):
    """SAM 2's cross-attention: keys of 3 frames turned on their grid (pointers at position 0, which does not turn them)
    through pages, the oldest frame's pages overwritten by a new one, against rope_attention on the gathered memory."""
    import sam_oracle as oracle

    side, d, page, dt = 16, 64, 64, torch.float16
    n, ptr = side * side, 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    cos, sin = (torch.from_numpy(t).cuda() for t in oracle.rope_tables(side, 1.0, d, 10000.0))
    at = torch.arange(n, device="cuda", dtype=torch.int32)
    grid = torch.stack([at % side, at // side], -1)
    freqs, axes = hip.rope_freqs((d // 4, d // 4))
    kp, vp = (torch.zeros(3 * n // page + 1, 1, page, d, device="cuda", dtype=dt) for _ in range(2))
    per = n // page
    frames = [(randn(gen, dt, n, 1, d), randn(gen, dt, n, 1, d)) for _ in range(4)]
    pointers = randn(gen, dt, ptr, 1, d), randn(gen, dt, ptr, 1, d)
    q = randn(gen, dt, n, 1, d)

    def write(k, v, pages, pos):
        k = hip.rope_axes(k, pos, freqs, axes)
        hip.kv_write(k, v, kp, vp, ints(*pages).view(1, -1), ints(0, k.shape[0]), ints(k.shape[0]))

    for i in range(3):
        write(*frames[i], range(i * per, (i + 1) * per), grid)
    write(*pointers, [3 * per], torch.zeros(ptr, 2, device="cuda", dtype=torch.int32))
    write(*frames[3], range(0, per), grid)  # over the oldest frame's pages
    order = [1, 2, 3]
    pages = [*range(per, 3 * per), *range(0, per), 3 * per]
    got = hip.paged_attention(hip.rope_axes(q, grid, freqs, axes), kp, vp, ints(*pages).view(1, -1), ints(0, n),
                              ints(3 * n + ptr), causal=False)
    k, v = (torch.cat([frames[i][j] for i in order] + [pointers[j]]).squeeze(1)[None] for j in range(2))
    want = hip.rope_attention(q.squeeze(1)[None], k, v, cos, sin, ptr)
    # both round q and k to f16 after the turn (tables off by 2^-24 * 15 radians at most: f16 neighbours, 2^-10 of a
    # value, on few of them), then P and the output: two outputs' roundings and two P's, of values up to 4
    assert (got.squeeze(1).float() - want[0].float()).abs().max() <= 4 * (2 * 2.0 ** -11 + 2 * 2.0 ** -11 + 2.0 ** -10)


@pytest.mark.parametrize("dtype, fp8, group", [("f16", True, 1), ("bf16", False, 4), ("f32", False, 2)])
def test_graphs_replay_as_eager_calls(hip, dtype, fp8, group):
    """Two graphs of one decoding step each (their own workspaces: splits that join), replayed in turn with eager work and
    synchronisations between, on tables, lengths and tokens that change from replay to replay."""
    dt, b, heads, d, page, width = DT[dtype], 3, 2, 128, 16, 300
    gen = torch.Generator(device="cuda").manual_seed(2)
    m = Memory(hip, b, heads, group, d, page, width, dt, fp8)
    starts = ints(0, 1, 2, 3)
    inputs = [[randn(gen, dt, b, heads * group, d), randn(gen, dt, b, heads, d), randn(gen, dt, b, heads, d),
               torch.zeros(b, 3, device="cuda", dtype=torch.int32), ints(1, 1, 1)] for _ in range(2)]

    def step(i):
        q, k, v, pos, lens = inputs[i]
        return m.step(q, k, v, pos, starts, lens, max_q=1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    side.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for r in range(5):
        for i in (0, 1) if r % 2 == 0 else (1, 0):
            q, k, v, pos, lens = inputs[i]
            for x in (q, k, v):
                x.copy_(randn(gen, dt, *x.shape))
            pos.random_(0, 1 << 16)
            lens.copy_(torch.randint(1, width * page, (b,)).to(torch.int32))
            m.table.copy_(m.table[:, torch.randperm(width, device="cuda")])
            graphs[i].replay()
            got = outs[i].clone()
            torch.cuda.synchronize()
            assert torch.equal(got, step(i))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_streams_side_by_side_and_repeated_bits(hip, dtype):
    """Calls on two streams at once (workspaces of their own) equal the calls one after the other, and a call repeats its
    bits, with splits and without."""
    dt = DT[dtype]
    gen = torch.Generator(device="cuda").manual_seed(3)
    jobs = []
    for lens, chunk in (((4000, 900), 1), ((700, 2000), 100)):
        m = Memory(hip, 2, 2, 4, 128, 16, 256, dt, False)
        full = randn(gen, dt, sum(lens), 2, 128), randn(gen, dt, sum(lens), 2, 128)
        hip.kv_write(*full, m.k, m.v, m.table, ints(0, lens[0], sum(lens)), ints(*lens))
        q = randn(gen, dt, 2 * chunk, 8, 128)
        jobs.append(lambda m=m, q=q, c=chunk, lens=lens: hip.paged_attention(q, m.k, m.v, m.table, ints(0, c, 2 * c), ints(*lens)))
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append([j() for _ in range(4)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, w) for x in g)


def test_a_long_cache_whose_offsets_pass_32_bits(hip):
    """A pool of 5 GiB whose used pages lie at its end: rows beyond 2^32 bytes are written, read and attended as near
    ones are."""
    heads, page, d, dt = 8, 64, 128, torch.float16
    pages = (5 << 30) // (heads * page * d * 2)
    far_pool = torch.empty(pages, heads, page, d, device="cuda", dtype=dt)
    near_pool = torch.empty(4, heads, page, d, device="cuda", dtype=dt)
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, q = randn(gen, dt, 200, heads, d), randn(gen, dt, 200, heads, d)  # values as keys too: one pool for both
    far, near = ints(pages - 1, pages - 4, pages - 2, pages - 3).view(1, 4), ints(3, 0, 1, 2).view(1, 4)
    st, ln = ints(0, 200), ints(200)
    hip.kv_write(x, x, far_pool, far_pool, far, st, ln)
    hip.kv_write(x, x, near_pool, near_pool, near, st, ln)
    read = hip.kv_read(far_pool, far_pool, far, ln, 200)
    assert torch.equal(read[0][0], x) and torch.equal(read[1][0], x)
    for rows in (q, q[:1]):
        s = ints(0, rows.shape[0])
        assert torch.equal(hip.paged_attention(rows, far_pool, far_pool, far, s, ln),
                           hip.paged_attention(rows, near_pool, near_pool, near, s, ln))
