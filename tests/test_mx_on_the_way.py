"""Which linear layers on few rows pack them on their way to the product: while a CU's workgroups pack 8192 values of a row in all."""
import os

import pytest
import torch

import sam_hip


@pytest.fixture(scope="module")
def size():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    return sam_hip.load().sam_hip_mx_linear_workspace_size


@pytest.mark.parametrize("m, n, k, on_the_way", [
    (16, 4096, 8192, True), (16, 4096, 8224, False), (17, 4096, 32, False), (1, 1, 8192, True),
    # up to 8 rows a workgroup takes 16 columns: 8192 columns are two workgroups a CU
    (8, 8192, 4096, True), (8, 8192, 4128, False), (8, 8192, 8192, False), (8, 16384, 2048, True), (8, 16384, 2080, False),
    # past that 32 where no CU gets more columns so
    (9, 8192, 8192, True), (16, 8192, 8192, True), (16, 8192, 8224, False), (9, 16384, 4096, True), (16, 16384, 4128, False),
    # 513 blocks of 16 columns are three a CU, in pairs four
    (16, 8200, 2720, True), (16, 8200, 4096, False), (16, 11000, 2720, True), (16, 11000, 2752, False)])
def test_what_a_cu_packs_in_all(size, m, n, k, on_the_way):
    assert size(m, n, k) == (0 if on_the_way else m * (k // 2 + k // 32))  # 256 CUs: an MI355X, and without a device


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m, n, k", [(9, 8192, 8192), (16, 8192, 8192), (16, 8191, 8160), (13, 4130, 8192), (16, 16384, 4096), (8, 8192, 8192), (16, 4096, 8192)])
def test_both_ways_agree(m, n, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(m + k)
    x, bias = torch.randn(m, k, generator=g, device="cuda").to(dtype), torch.randn(n, generator=g, device="cuda").to(dtype)
    w = sam_hip.mx_pack(torch.randn(n, k, generator=g, device="cuda"))
    assert torch.equal(sam_hip.mx_linear(x, *w, bias, gelu=True), sam_hip.mx_matmul(*sam_hip.mx_pack(x), *w, bias, gelu=True, dtype=dtype))
