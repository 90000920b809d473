"""The 4-bit numbers' C entry points refuse bad arguments before touching a GPU (CPU only: no kernel is launched), and the
reference that the GPU tests use keeps its own promises."""
import ctypes
import os
import re

import pytest
import torch

import mx_ref as ref
import sam_hip

vp = ctypes.c_void_p
FAKE = vp(0x1000)  # never dereferenced: every call below fails first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    return sam_hip.load()


def pack(lib, x=FAKE, codes=FAKE, scales=FAKE, dtype=1, rows=4, k=64):
    return lib.sam_hip_mx_pack(x, codes, scales, dtype, rows, k, None)


def unpack(lib, x=FAKE, codes=FAKE, scales=FAKE, dtype=1, rows=4, k=64):
    return lib.sam_hip_mx_unpack(codes, scales, x, dtype, rows, k, None)


def matmul(lib, a=FAKE, sa=FAKE, b=FAKE, sb=FAKE, bias=None, out=FAKE, dtype=1, m=4, n=4, k=64, gelu=0):
    return lib.sam_hip_mx_matmul(a, sa, b, sb, bias, out, dtype, m, n, k, gelu, None)


def linear(lib, x=FAKE, w=FAKE, sw=FAKE, bias=None, out=FAKE, dtype=1, m=4, n=4, k=64, ws=FAKE, ws_bytes=1 << 20):
    return lib.sam_hip_mx_linear(x, w, sw, bias, out, dtype, m, n, k, 0, ws, ws_bytes, None)


@pytest.mark.parametrize("change, code", [
    ({"x": None}, 1), ({"w": None}, 1), ({"sw": None}, 1), ({"out": None}, 1), ({"dtype": 3}, 2), ({"m": -1}, 1), ({"n": -1}, 1),
    ({"k": 40}, 1), ({"k": (1 << 22) + 32}, 3), ({"m": 1 << 15, "k": 1 << 22, "n": 1}, 3), ({"x": vp(0x1008)}, 3), ({"w": vp(0x1008)}, 3),
    ({"ws": None, "m": 17}, 1), ({"ws": vp(0x1008)}, 3), ({"m": 17, "ws_bytes": 17 * 34 - 1}, 1), ({"bias": vp(0x1008)}, 3), ({"out": vp(0x1008)}, 3)])
def test_linear_refuses(lib, change, code):
    assert linear(lib, **change) == code
    assert lib.sam_hip_last_error()


def test_linear_workspace(lib):
    size = lib.sam_hip_mx_linear_workspace_size
    assert size(17, 9, 64) == 17 * 34 and size(16, 9, 1 << 20) == 16 * (34 << 14) and size(16, 4096, 8192) == size(0, 9, 64) == size(99, 0, 64) == 0
    assert size(3, 9, 48) == size(-1, 9, 64) == size(1 << 15, 1, 1 << 22) == -1 and linear(lib, m=0) == 0


@pytest.mark.parametrize("call", [pack, unpack])
@pytest.mark.parametrize("change, code", [
    ({"x": None}, 1), ({"codes": None}, 1), ({"scales": None}, 1), ({"dtype": 3}, 2), ({"dtype": -1}, 2), ({"rows": -1}, 1),
    ({"k": 0}, 1), ({"k": 48}, 1), ({"k": -32}, 1), ({"rows": 1 << 31}, 3), ({"rows": 1 << 30, "k": 32}, 3), ({"x": vp(0x1008)}, 3),
    ({"codes": vp(0x1004)}, 3)])
def test_pack_and_unpack_refuse(lib, call, change, code):
    assert call(lib, **change) == code
    assert lib.sam_hip_last_error()


@pytest.mark.parametrize("change, code", [
    ({"a": None}, 1), ({"sa": None}, 1), ({"b": None}, 1), ({"sb": None}, 1), ({"out": None}, 1), ({"dtype": 3}, 2), ({"m": -1}, 1),
    ({"n": -1}, 1), ({"k": 0}, 1), ({"k": 40}, 1), ({"k": (1 << 22) + 32}, 3), ({"m": 1 << 20, "n": 1 << 16}, 3),
    ({"m": (1 << 30) + 1, "n": 1}, 3), ({"m": 1, "n": (1 << 25) + 1}, 3), ({"m": 1 << 30, "n": 1}, 3), ({"a": vp(0x1008)}, 3),
    ({"b": vp(0x1008)}, 3), ({"out": vp(0x1002)}, 3), ({"bias": vp(0x1008)}, 3)])
def test_matmul_refuses(lib, change, code):
    assert matmul(lib, **change) == code
    assert lib.sam_hip_last_error()


def test_the_header_declares_what_the_library_exports(lib):
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "sam_hip_mx.h")).read()
    names = set(re.findall(r"\b(sam_hip_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == {"sam_hip_mx_pack", "sam_hip_mx_unpack", "sam_hip_mx_matmul", "sam_hip_mx_linear", "sam_hip_mx_linear_workspace_size"}
    assert all(hasattr(lib, n) for n in names)


def test_the_switch_covers_them(lib):
    lib.sam_hip_set_enabled(0)
    try:
        assert pack(lib, x=None) == unpack(lib, x=None) == matmul(lib, a=None) == linear(lib, x=None) == 5
    finally:
        lib.sam_hip_set_enabled(1)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.float16)
    codes, scale = torch.zeros(2, 32, dtype=torch.uint8).view(torch.float4_e2m1fn_x2), torch.zeros(2, 2, dtype=torch.uint8)
    for call in (lambda: sam_hip.mx_pack(x), lambda: sam_hip.mx_unpack(codes, scale), lambda: sam_hip.mx_matmul(codes, scale, codes, scale),
                 lambda: sam_hip.mx_linear(x, codes, scale)):
        with pytest.raises(sam_hip.SamHipError, match="device tensors"):
            call()


def test_reference_quantiser_rounds_to_the_nearest():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 96, generator=g, dtype=torch.float64) * torch.pow(10.0, torch.randint(-3, 4, (64, 1), generator=g).double())
    x[0], x[1, 0], x[2, 90] = 0.0, float("inf"), float("nan")
    val, codes, s = ref.quantise(x)
    assert torch.equal(torch.nan_to_num(ref.values(ref.packed(codes), s), -1.0), torch.nan_to_num(val, -1.0))
    assert s[0].tolist() == [127] * 3 and s[1, 0] == 255 and s[1, 1] != 255 and s[2, 2] == 255
    grid = torch.tensor(ref.GRID, dtype=torch.float64)
    for r in range(3, 64):
        for b in range(3):
            v, y, two = val[r, 32 * b:32 * b + 32], x[r, 32 * b:32 * b + 32], 2.0 ** (int(s[r, b]) - 127)
            assert 3 * two < y.abs().max() <= 6 * two
            assert torch.equal((v.abs() / two - y.abs() / two).abs(), (y.abs()[:, None] / two - grid).abs().min(-1).values)
    tie = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4, dtype=torch.float64)
    assert ref.quantise(tie)[0][:8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]


def test_the_paged_memory_refuses_what_4_bits_cannot_hold(lib):
    from test_paged_abi import attend, read, write

    for call in (write, read, attend):
        for change, code in (({"cache": 4, "d": 72}, 3), ({"cache": 4, "d": 80}, 3), ({"cache": 4, "ks": None}, 1), ({"cache": 4, "vs": None}, 1),
                             ({"cache": 5}, 2), ({"cache": 4, "dtype": 3}, 2), ({"cache": 4, "k_pages": vp(0x1008)}, 3)):
            assert call(lib, **change) == code
            assert lib.sam_hip_last_error()
    size = lib.sam_hip_paged_attention_workspace_size
    assert size(1, 4, 1, 1, 8, 1, 128, 1, 1 << 16) > 0 and size(1, 5, 1, 1, 8, 1, 128, 1, 64) == -1
