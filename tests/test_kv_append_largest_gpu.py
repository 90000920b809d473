"""Keys whose turn is beyond f32's largest number are infinite, as rope_axes gives them to kv_write."""
import math

import pytest
import torch

from test_kv_append_gpu import DT, a_pool, same_bytes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairs, partner", [("adjacent", 1), ("halves", 1)])  # one pair: both layouts turn columns 0 and 1
def test_a_turn_past_the_largest_number(hip, held, dtype, pairs, partner):
    dt = DT[dtype]
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    k = torch.randn(4, 1, 64, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(dt)
    k[0, 0, 0], k[0, 0, partner] = 3.3e38, 2.3e38    # the second becomes 3.96e38
    k[1, 0, 0], k[1, 0, partner] = -3.3e38, -2.3e38
    k[2, 0, 0], k[2, 0, partner] = 2.3e38, 1.3e38    # 2.55e38: finite
    turned = k.double()
    c = math.sqrt(0.5)
    a, b = turned[..., 0].clone(), turned[..., partner].clone()
    turned[..., 0], turned[..., partner] = (a - b) * c, (a + b) * c
    want_k = turned.float()  # what is beyond f32 is infinite; rounded again to bf16, where no sum of this test is near a border
    assert torch.isinf(want_k).sum() == 2
    freqs, axes = torch.tensor([math.pi / 4], dtype=torch.float64, device="cuda"), i(0)
    new, old = (a_pool(held, 1, 1, 4, 64, dt) for _ in range(2))
    hip.kv_append(None, k, k, freqs, axes, new[0], new[1], i(0).view(1, 1), i(0, 4), i(4), new[2], new[3], torch.ones(4, 1, device="cuda").int(), pairs)
    if held == "own":
        want = want_k.to(dt)
        hip.kv_write(want, k, old[0], old[1], i(0).view(1, 1), i(0, 4), i(4))
    else:
        wide = a_pool(held, 1, 1, 4, 64, torch.float32)
        hip.kv_write(want_k, k.float(), wide[0], wide[1], i(0).view(1, 1), i(0, 4), i(4), wide[2], wide[3])
        old = wide
    for x, y in zip(new, old):
        assert x is None or same_bytes(x, y)
    if held != "own":
        back, _ = hip.kv_read(new[0], new[1], i(0).view(1, 1), i(4), 4, new[2], new[3], dtype=torch.float32)
        assert torch.isnan(back[0, :2, 0, partner]).all() and torch.isfinite(back[0, 2:]).all()
