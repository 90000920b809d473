"""The image encoder with its blocks' linears in 4 bits (sam_encoder.pack_linears) on an MI355X."""
import pytest
import torch

import mx_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def enc():
    import sam_encoder
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_encoder


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [160, 128])
def test_a_packed_block_is_its_own_steps(enc, dim, dtype):
    """A block's linears are the products of packed rows and packed weights, within the bound of their f32 sums; the rest
    of the block is what it is with other weights."""
    import sam_hip as hip

    cfg = enc.EncoderConfig(dim, 1, 2, (), img_size=448)
    w = enc.random_weights(cfg, dtype=dtype, seed=3, std=0.05)
    packed = enc.pack_linears(w)
    p, q = w.blocks[0], packed.blocks[0]
    assert isinstance(p.qkv_w, torch.Tensor) and q.norm1_w is p.norm1_w and packed.pos is w.pos
    x = torch.randn(1, 28, 28, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    rows = x.reshape(784, dim)
    for name in ("qkv_w", "proj_w"):
        got = enc.linear(rows, getattr(q, name))
        want, bound = mx_ref.product(mx_ref.quantise(rows.cpu())[0], mx_ref.quantise(getattr(p, name).cpu())[0], None, False, dtype)
        assert ((got.cpu().double() - want).abs() <= bound).all()
    xn = torch.nn.functional.layer_norm(x, (dim,), q.norm1_w, q.norm1_b, 1e-6)
    got, _ = enc.block(x, xn, q, cfg.heads)
    y, xn2 = hip.bias_residual_ln(x, enc.attention(xn, q, cfg.heads), q.proj_b, q.norm2_w, q.norm2_b, 1e-6)
    m = hip.mx_linear(xn2.reshape(784, dim), *hip.mx_pack(p.lin1_w), p.lin1_b, gelu=True)
    assert torch.equal(got, hip.bias_residual(y, hip.mx_linear(m, *hip.mx_pack(p.lin2_w)).view(1, 28, 28, dim), q.lin2_b))


def test_a_packed_encoder_runs(enc):
    cfg = enc.EncoderConfig(160, 2, 2, (1,))
    w = enc.pack_linears(enc.random_weights(cfg, seed=3, std=0.05))
    img = torch.randn(1, 3, 1024, 1024, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").half()
    out = enc.encoder_forward(img, w)
    assert out.shape == (1, 256, 64, 64) and torch.isfinite(out).all()
    assert torch.equal(enc.encoder_forward(img, w), out)
