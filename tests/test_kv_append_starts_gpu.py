"""kv_append under starts that do not ascend: which tokens a sequence takes is what kv_write takes, and the queries of the
others are 0."""
import random

import pytest
import torch

from test_kv_append_gpu import a_pool, same_bytes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import sam_hip

    sam_hip.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return sam_hip


def of_a_sequence(starts, t):
    """Whether token t is one of the sequence that the ends at or before it lead to."""
    b = sum(e <= t for e in starts[1:])
    return b < len(starts) - 1 and starts[b] <= t < starts[b + 1]


def random_starts(n):
    r = random.Random(n)
    return [r.randint(-2, 24) for _ in range(n + 1)]


STARTS = [[0, 9, 9, 2], [0, 5, 3, 12, 12], [4, 2, 8, 12], [0, 12, 6, 6], [24, 0, 24], [0, 24, 24, 23], *(random_starts(n) for n in (2, 5, 9, 40, 64, 65, 90))]


@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
@pytest.mark.parametrize("heads, d", [(1, 64), (3, 64), (2, 128), (1, 256)])
@pytest.mark.parametrize("starts", STARTS, ids=str)
def test_tokens_of_starts_that_do_not_ascend(hip, held, heads, d, starts):
    tokens, batch, page = 24, len(starts) - 1, 16
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(batch)
    q, k, v = (torch.randn(tokens, h, d, generator=g, device="cuda").half() for h in (2 * heads, heads, heads))
    freqs, axes = torch.zeros(0, dtype=torch.float64, device="cuda"), i([])
    table = torch.arange(3 * batch, device="cuda").int().view(batch, 3)  # no two sequences share a page
    lens = i([40] * batch)
    a, b = (a_pool(held, 3 * batch, heads, page, d, torch.float16) for _ in range(2))
    for x in (*a, *b):
        if x is not None:
            x.view(torch.uint8).zero_()
    got = hip.kv_append(q, k, v, freqs, axes, a[0], a[1], table, i(starts), lens, a[2], a[3])
    hip.kv_write(k, v, b[0], b[1], table, i(starts), lens, b[2], b[3])
    for x, y in zip(a, b):
        assert x is None or same_bytes(x, y)
    known = torch.tensor([of_a_sequence(starts, t) for t in range(tokens)], device="cuda")
    assert torch.equal(got, torch.where(known[:, None, None], q, torch.zeros_like(q)))
