"""rope_axes on an MI355X against the definition in 64 bits, with the bound of its roundings (paged_ref.rope_bound)."""
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


def check(got, x, pos, freqs, axes, pairs, inverse=False):
    want = ref.rope(x.cpu(), pos.cpu(), freqs.cpu(), axes.cpu(), pairs, inverse)
    off = (got.cpu().double() - want).abs()
    over = (off - ref.rope_bound(x.cpu(), want, len(freqs), pairs, x.dtype)).max()
    assert over <= 0, f"{over:.3g} past the bound, {off.max():.3g} off"


CASES = [  # B, L, H, D, sections
    (1, 1, 1, 8, (2, 2)), (1, 1, 8, 64, (8, 12, 12)), (2, 37, 3, 80, (10, 30)), (1, 300, 1, 256, (32, 48, 48)),
    (3, 5, 16, 72, (36,)), (1, 64, 5, 128, (16, 8, 8, 16)), (2, 9, 2, 30, (7, 3)), (1, 513, 6, 96, (5, 6)),
    (1, 2000, 20, 64, (16, 16)), (1, 3, 2, 40, (0, 8))]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("shape", CASES)
def test_matches_the_definition(hip, dtype, pairs, shape):
    b, l, h, d, sections = shape
    g = torch.Generator(device="cuda").manual_seed(l + d)
    x = torch.randn(b, l, h, d, generator=g, device="cuda").to(DT[dtype])
    pos = torch.randint(0, 1 << 20, (b, l, len(sections)), generator=g, device="cuda", dtype=torch.int32)
    freqs, axes = hip.rope_freqs(sections)
    check(hip.rope_axes(x, pos, freqs, axes, pairs=pairs), x, pos, freqs, axes, pairs)
    check(hip.rope_axes(x, pos, freqs, axes, pairs=pairs, inverse=True), x, pos, freqs, axes, pairs, True)


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_far_and_negative_positions(hip, pairs):
    x = torch.randn(1, 7, 2, 64, device="cuda")
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, -12345], device="cuda", dtype=torch.int32)
    pos = torch.stack([pos, pos.flip(0)], -1)[None]
    freqs, axes = hip.rope_freqs((16, 16), theta=10000.0)
    check(hip.rope_axes(x, pos, freqs, axes, pairs=pairs), x, pos, freqs, axes, pairs)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_strides_views_shared_positions_and_in_place(hip, dtype, pairs):
    g = torch.Generator(device="cuda").manual_seed(5)
    freqs, axes = hip.rope_freqs((8, 8, 16))
    packed = torch.randn(2, 50, 3, 4, 64, generator=g, device="cuda").to(DT[dtype])
    pos = torch.randint(0, 4000, (50, 3), generator=g, device="cuda", dtype=torch.int32)
    wide = pos.expand(2, 50, 3)
    for x in (packed[:, :, 1], packed[:, ::2, 0], packed[..., 0, :, :].transpose(1, 2)[..., :, 1:3, :].transpose(1, 2)):
        p = pos[: x.shape[1]]
        check(hip.rope_axes(x, p, freqs, axes, pairs=pairs), x, wide[:, : x.shape[1]], freqs, axes, pairs)
    odd = torch.randn(2 * 50 * 4 * 64 + 1, generator=g, device="cuda").to(DT[dtype])[1:].view(2, 50, 4, 64)  # off 16 bytes
    check(hip.rope_axes(odd, pos, freqs, axes, pairs=pairs), odd, wide, freqs, axes, pairs)
    flat = packed[0, :, 1]
    assert torch.equal(hip.rope_axes(flat, pos, freqs, axes, pairs=pairs), hip.rope_axes(packed[:1, :, 1], pos, freqs, axes, pairs=pairs)[0])
    want, rest = hip.rope_axes(packed[:, :, 1], pos, freqs, axes, pairs=pairs), packed.clone()
    back = hip.rope_axes(packed[:, :, 1], pos, freqs, axes, pairs=pairs, out=packed[:, :, 1])
    assert torch.equal(back, want) and torch.equal(packed[:, :, 0], rest[:, :, 0]) and torch.equal(packed[:, :, 2], rest[:, :, 2])


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_gradient_is_the_inverse_turn(hip, pairs):
    """y = R x is linear, so dL/dx = R^T dL/dy: against <R^T w, e> = <w, R e> for unit steps e, which are differences of
    the forward pass (exact for a linear map up to its roundings, 4e-7 of |x0| + |x1| = 1 each)."""
    freqs, axes = hip.rope_freqs((5, 3))
    pos = torch.randint(0, 1000, (1, 6, 2), device="cuda", dtype=torch.int32)
    w = torch.randn(1, 6, 1, 20, device="cuda")
    grad = hip.rope_axes(w, pos, freqs, axes, pairs=pairs, inverse=True)
    for c in range(20):
        e = torch.zeros(1, 6, 1, 20, device="cuda")
        e[..., c] = 1.0
        by_difference = (hip.rope_axes(e, pos, freqs, axes, pairs=pairs).double() * w.double()).sum(-1)
        assert (grad[..., c].double() - by_difference).abs().max() <= 2 * 4e-7 * 2 * w.abs().max()


def test_matches_the_two_axis_tables(hip):
    """On a grid, the positions (column, row) give the rotation that sam_hip.rope applies from its f32 tables, to the
    tables' own rounding (angles of up to 63 rounded to f32: 63 * 2^-24 = 3.8e-6)."""
    import sam_oracle as oracle

    side, d = 64, 256
    cos, sin = (torch.from_numpy(t).cuda() for t in oracle.rope_tables(side, 1.0, d, 10000.0))
    x = torch.randn(1, side * side, d, device="cuda")
    at = torch.arange(side * side, device="cuda", dtype=torch.int32)
    pos = torch.stack([at % side, at // side], -1)
    freqs, axes = hip.rope_freqs((d // 4, d // 4))
    got = hip.rope_axes(x.unsqueeze(2), pos, freqs, axes).squeeze(2)
    assert (got - hip.rope(x, cos, sin)).abs().max() <= (2 * 3.8e-6 + 4e-7) * 2 * x.abs().max()


def test_empty_calls_and_refusals(hip):
    freqs, axes = hip.rope_freqs((16, 16))
    x = torch.randn(1, 4, 2, 64, device="cuda")
    pos = torch.zeros(1, 4, 2, device="cuda", dtype=torch.int32)
    assert hip.rope_axes(x[:, :0], pos[:, :0], freqs, axes).shape == (1, 0, 2, 64)
    none = (freqs[:0], axes[:0])
    assert torch.equal(hip.rope_axes(x, pos, *none), x)
    bad_axis = axes.clone()
    bad_axis[:] = 7  # no such axis: position 0
    assert torch.equal(hip.rope_axes(x, pos + 5, freqs, bad_axis), x)
    for call in (lambda: hip.rope_axes(x, pos.long(), freqs, axes), lambda: hip.rope_axes(x, pos, freqs.float(), axes),
                 lambda: hip.rope_axes(x, pos, freqs, axes[:-1]), lambda: hip.rope_axes(x, pos[:, :3], freqs, axes),
                 lambda: hip.rope_axes(x[..., :32], pos, freqs, axes), lambda: hip.rope_axes(x, pos, freqs, axes, pairs="x"),
                 lambda: hip.rope_axes(x, pos, freqs, axes, out=x.half()), lambda: hip.rope_axes(x.double(), pos, freqs, axes),
                 lambda: hip.rope_axes(x[0, 0], pos, freqs, axes), lambda: hip.rope_axes(x, pos.cpu(), freqs, axes)):
        with pytest.raises(hip.SamHipError):
            call()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("naxes", [1, 4, 5])
@pytest.mark.parametrize("shape, off", [((2, 5, 3, 64), 0), ((1, 9000, 8, 128), 0), ((2, 5, 3, 30), 0), ((2, 5, 3, 64), 1)])
def test_no_pairs_need_no_positions(hip, dtype, naxes, shape, off):
    """The C entry takes NULL for pos, freqs and axes where pairs is 0: out becomes a copy of x, with vectors and without."""
    b, l, h, d = shape
    x = torch.randn(b * l * h * d + off, device="cuda").to(DT[dtype])[off:].view(shape)
    out = torch.zeros_like(x)
    code = {"f32": 0, "f16": 1, "bf16": 2}[dtype]
    for halves in (0, 1):
        out.zero_()
        rc = hip.load().sam_hip_rope_axes(x.data_ptr(), None, None, None, out.data_ptr(), code, b, l, h, d, 0, naxes, None, None,
                                          None, halves, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(out, x)
