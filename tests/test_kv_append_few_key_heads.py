"""kv_append with fewer key heads than a thread takes of one token: the choice, and results against the definition."""
import ctypes
import os

import pytest
import torch

import sam_hip
import test_kv_append_gpu as t


@pytest.fixture(scope="module")
def heads_of():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    # samhip::kv_append_heads(int bytes of an element, int tokens, int heads, int kv_heads, int d)
    fn = ctypes.CDLL(sam_hip.LIB_PATH)._ZN6samhip15kv_append_headsEiiiii
    fn.argtypes, fn.restype = [ctypes.c_int] * 5, ctypes.c_int
    return fn


def test_the_larger_count_of_heads_decides(heads_of):
    for kv in (1, 2, 3, 4, 8):
        assert heads_of(2, 16384, 16, kv, 128) == 4 and heads_of(4, 16384, 16, kv, 128) == 2
        assert heads_of(2, 16, 16, kv, 128) == 1 and heads_of(4, 16, 16, kv, 128) == 1
    assert heads_of(2, 16384, 1, 1, 256) == heads_of(4, 16384, 1, 1, 256) == heads_of(2, 16384, 2, 2, 128) == 1
    assert heads_of(2, 65536, 0, 4, 128) == 4 and heads_of(2, 65536, 0, 1, 128) == 1  # no queries
    assert heads_of(2, 960, 16, 1, 128) == 1 and heads_of(2, 1024, 16, 1, 128) == 4
    assert heads_of(2, (1 << 27) // 65536 - 1, 65535, 1, 256) == 4  # the most rows of a call


FEW = [([1700, 300], [1800, 900], 16, 1, 128, 16, 64, 0), ([2100], [2100], 7, 2, 96, 24, 45, 3), ([2800, 7], [2900, 8], 9, 3, 64, 8, 20, 1),
       ([1500], [1537], 5, 1, 256, 64, 128, 2), ([1200], [1200], 13, 3, 160, 16, 0, 1), ([5600], [5600], 4, 2, 64, 32, 13, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("held", ["own", "e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("case", FEW, ids=[f"{c[2]}-{c[3]}-{c[4]}" for c in FEW])
def test_matches_the_definition(heads_of, held, dtype, pairs, case):
    chunks, _, hq, hkv, d, *_ = case
    if not (held == "e2m1" and d % 32):
        assert heads_of(4 if dtype == "f32" else 2, sum(chunks), hq, hkv, d) > 1
        t.test_matches_the_definition(sam_hip, held, dtype, pairs, case)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hq, hkv", [(5, 1), (7, 3), (16, 2)])
def test_in_place(hq, hkv, dtype):
    """Queries turned in their own place are those turned into another: a thread's last heads may be another's."""
    g = torch.Generator(device="cuda").manual_seed(0)
    n, d = 4000, 128
    q, k = (torch.randn(n, h, d, generator=g, device="cuda").to(dtype) for h in (hq, hkv))
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    freqs, axes = sam_hip.rope_freqs((d // 2,))
    kp, vp = (torch.zeros(1, hkv, n, d, device="cuda", dtype=dtype) for _ in range(2))
    call = lambda q, **kw: sam_hip.kv_append(q, k, k, freqs, axes, kp, vp, i(0).view(1, 1), i(0, n), i(n), **kw)
    for pairs in ("adjacent", "halves"):
        want = call(q, pairs=pairs)
        for _ in range(3):
            own = q.clone()
            assert call(own, pairs=pairs, out=own) is own and torch.equal(own, want)
