"""A whole encoder with packed linears (sam_encoder.pack_linears): every linear and no other is the product of packed rows and
packed weights, and what 4 bits cost on random weights stays within their roundings."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def enc():
    import sam_encoder
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_encoder


def image(size, batch, dtype):
    return torch.randn(batch, 3, size, size, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(dtype)


@pytest.mark.parametrize("dim, heads, depth, glob", [(160, 2, 3, (1,)), (128, 2, 2, ())])
def test_it_is_the_encoder_with_its_linears_packed(enc, monkeypatch, dim, heads, depth, glob):
    """The plain encoder's forward with F.linear put in place by packing both operands, for the blocks' weights alone: in f32 the
    same bits, as bias and GELU are the same sums beside the product and within it."""
    import sam_hip as hip

    cfg = enc.EncoderConfig(dim, depth, heads, glob, img_size=448)
    w = enc.random_weights(cfg, dtype=torch.float32, seed=3, std=0.05)
    img = image(448, 2, torch.float32)
    got = enc.encoder_forward(img, enc.pack_linears(w))
    of_blocks = {t.data_ptr() for p in w.blocks for t in (p.qkv_w, p.proj_w, p.lin1_w, p.lin2_w)}
    calls = []

    def linear(x, weight):
        if weight.data_ptr() not in of_blocks:
            return torch.nn.functional.linear(x, weight)
        calls.append(weight.data_ptr())
        return hip.mx_matmul(*hip.mx_pack(x), *hip.mx_pack(weight))

    monkeypatch.setattr(enc, "F", types.SimpleNamespace(**{**vars(torch.nn.functional), "linear": linear}))
    want = enc.encoder_forward(img, w)
    assert len(calls) == 4 * depth and set(calls) == of_blocks
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_4_bits_cost_on_random_weights(enc, dtype):
    """A value of a block is off by at most half a step, a quarter of it (an even spread over that is 0.145 of it), or by a quarter
    of a scale that is a third of the block's largest at most: below 0.145 of the values together. Both operands' errors are
    independent: 0.205 of a product. Two products follow one another in each half of a block (the GELU between lets 1.13 of an
    error through): 0.31 of what the half adds to the residual. The neck keeps proportions. So the outputs differ by 0.31 of
    their size at most, and by more than 16 bits' own roundings; of two encoders with other weights by 1.41."""
    cfg = enc.EncoderConfig(160, 2, 2, (1,), img_size=448)
    w = enc.random_weights(cfg, dtype=dtype, seed=3, std=0.05)
    img = image(448, 1, dtype)
    plain, packed, other = (enc.encoder_forward(img, x).double() for x in (w, enc.pack_linears(w), enc.random_weights(cfg, dtype=dtype, seed=4, std=0.05)))
    size = plain.norm()
    off = float((packed - plain).norm() / size)
    print("relative error", off)
    assert 2.0 ** -8 < off < 0.31 < float((other - plain).norm() / size)
