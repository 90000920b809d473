"""The tiles of the 4-bit product: sizes that the entry points take fit a launch, which counts threads in 32 bits."""
import ctypes
import os

import pytest
import torch

import sam_hip

THREADS = {64: 256, 128: 256, 256: 512}


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    return sam_hip.load()


def accepted(m, n, k):
    """The limits of include/sam_hip_mx.h."""
    return m * n < 1 << 36 and m <= 1 << 30 and n <= 1 << 25 and k <= 1 << 22 and -(-m // 128) * -(-n // 128) < 1 << 23


def test_every_accepted_size_fits_a_launch(lib):
    tile_of = ctypes.CDLL(sam_hip.LIB_PATH)._ZN6samhip15mx_product_tileEiiii  # samhip::mx_product_tile(int cus, int m, int n, int k)
    tile_of.argtypes, tile_of.restype = [ctypes.c_int] * 4, ctypes.c_int
    sizes = [33, 64, 65, 128, 160, 300, 1000, *(1 << b for b in range(11, 31)), *(3 << b for b in range(11, 29)), 420_000_000, (1 << 30) - 128,
             (1 << 30) - 511, (1 << 30) - 700, (1 << 29) - 1, 5 << 27]
    seen = set()
    for cus in (1, 80, 256, 304):
        for m in sizes:
            for n in [1, 16, 64, *sizes]:
                for k in (32, 256, 1024, 1 << 22):
                    if not accepted(m, n, k):
                        continue
                    t = tile_of(cus, m, n, k)
                    seen.add(t)
                    workgroups = (-(-m // t) * -(-n // t) + 7) // 8 * 8  # one share of them for each of eight XCDs
                    assert workgroups * THREADS[t] < 1 << 32, (cus, m, n, k, t)
    assert seen == {64, 128, 256}


@pytest.mark.gpu
def test_the_most_rows():
    """2^30 - 200 rows of 32 values to 2 columns, against the same rows 2^20 at a time."""
    m, n, part = (1 << 30) - 200, 2, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(0)
    codes = torch.randint(0, 256, (m, 16), generator=g, device="cuda", dtype=torch.uint8).view(torch.float4_e2m1fn_x2)
    scale = torch.randint(120, 134, (m, 1), generator=g, device="cuda", dtype=torch.uint8)
    w = sam_hip.mx_pack(torch.randn(n, 32, generator=g, device="cuda"))
    got = sam_hip.mx_matmul(codes, scale, *w, dtype=torch.float16)
    for i in range(0, m, part):
        assert torch.equal(got[i:i + part], sam_hip.mx_matmul(codes[i:i + part], scale[i:i + part], *w, dtype=torch.float16)), i
