"""The paged memory's C entry points refuse bad arguments before touching a GPU (CPU only: no kernel is launched),
and the reference that the GPU tests use keeps its own promises."""
import ctypes
import os
import re

import pytest
import torch

import paged_ref as ref
import sam_hip

vp, i, f, lp = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.POINTER(ctypes.c_long)
FAKE = vp(0x1000)  # never dereferenced: every call below fails first
E4M3 = 3


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    return sam_hip.load()


def strides(*s):
    return (ctypes.c_long * len(s))(*s)


def rope(lib, x=FAKE, pos=FAKE, freqs=FAKE, axes=FAKE, out=vp(0x2000), dtype=1, b=1, l=4, h=2, d=64, pairs=32, naxes=3,
         sx=None, sp=None, so=None):
    return lib.sam_hip_rope_axes(x, pos, freqs, axes, out, dtype, b, l, h, d, pairs, naxes, sx, sp, so, 0, 0, None)


@pytest.mark.parametrize("change, code", [
    ({"x": None}, 1), ({"pos": None}, 1), ({"freqs": None}, 1), ({"axes": None}, 1), ({"out": None}, 1),
    ({"dtype": 3}, 2), ({"dtype": -1}, 2), ({"b": -1}, 1), ({"h": 0}, 1), ({"pairs": -1}, 1), ({"pairs": 33}, 1),
    ({"naxes": 0}, 1), ({"b": 1 << 20, "l": 1 << 20}, 3), ({"x": vp(0x1001)}, 3), ({"freqs": vp(0x1004)}, 3),
    ({"sx": strides(512, -128, 64)}, 3), ({"out": FAKE, "sx": strides(512, 128, 64), "so": strides(1024, 256, 64)}, 1)])
def test_rope_axes_refuses(lib, change, code):
    assert rope(lib, **change) == code
    assert lib.sam_hip_last_error()


POOL = dict(k_pages=FAKE, v_pages=FAKE, ks=FAKE, vs=FAKE, table=FAKE, lens=FAKE, dtype=1, cache=1, batch=2, pages=8,
            kv_heads=2, page=16, d=64, width=4)


def write(lib, k=FAKE, v=FAKE, starts=FAKE, tokens=4, sk=None, sv=None, **change):
    a = {**POOL, **change}
    return lib.sam_hip_kv_write(k, v, a["k_pages"], a["v_pages"], a["ks"], a["vs"], a["table"], starts, a["lens"],
                                a["dtype"], a["cache"], tokens, a["batch"], a["pages"], a["kv_heads"], a["page"], a["d"],
                                a["width"], sk, sv, None)


def read(lib, k=FAKE, v=FAKE, max_len=64, **change):
    a = {**POOL, **change}
    return lib.sam_hip_kv_read(k, v, a["k_pages"], a["v_pages"], a["ks"], a["vs"], a["table"], a["lens"], a["dtype"],
                               a["cache"], a["batch"], max_len, a["pages"], a["kv_heads"], a["page"], a["d"], a["width"],
                               None)


def attend(lib, q=FAKE, out=FAKE, starts=FAKE, tokens=4, heads=4, sq=None, so=None, scale=0.1, max_q=4, max_len=64,
           ws=None, ws_bytes=0, **change):
    a = {**POOL, **change}
    return lib.sam_hip_paged_attention(q, a["k_pages"], a["v_pages"], a["ks"], a["vs"], a["table"], starts, a["lens"], out,
                                       a["dtype"], a["cache"], tokens, a["batch"], heads, a["pages"], a["kv_heads"],
                                       a["page"], a["d"], a["width"], sq, so, scale, 1, 0, max_q, max_len, ws, ws_bytes,
                                       None)


BAD_POOL = [({"k_pages": None}, 1), ({"v_pages": None}, 1), ({"table": None}, 1), ({"lens": None}, 1), ({"dtype": 4}, 2),
            ({"dtype": 1, "cache": 2}, 2), ({"dtype": 0, "cache": 1}, 2), ({"cache": E4M3, "ks": None}, 1),
            ({"cache": E4M3, "vs": None}, 1), ({"batch": 0}, 1), ({"pages": 0}, 1), ({"kv_heads": 0}, 1),
            ({"page": 0}, 1), ({"d": 0}, 1), ({"width": 0}, 1), ({"d": 20}, 3), ({"d": 264}, 3),
            ({"width": 1 << 20, "page": 1 << 10}, 3), ({"k_pages": vp(0x1008)}, 3)]


@pytest.mark.parametrize("call", [write, read, attend])
@pytest.mark.parametrize("change, code", BAD_POOL)
def test_bad_pools_are_refused(lib, call, change, code):
    extra = {"heads": 4 * max(1, change.get("kv_heads", 2))} if call is attend else {}
    assert call(lib, **extra, **change) == code
    assert lib.sam_hip_last_error()


@pytest.mark.parametrize("change, code", [
    ({"k": None}, 1), ({"v": None}, 1), ({"starts": None}, 1), ({"tokens": -1}, 1), ({"sk": strides(100, 64)}, 3),
    ({"sv": strides(-128, 64)}, 3), ({"k": vp(0x1002)}, 3)])
def test_kv_write_refuses(lib, change, code):
    assert write(lib, **change) == code


@pytest.mark.parametrize("change, code", [({"k": None}, 1), ({"v": None}, 1), ({"max_len": -1}, 1),
                                          ({"max_len": 0x7fffffff}, 3), ({"v": vp(0x1008)}, 3)])
def test_kv_read_refuses(lib, change, code):
    assert read(lib, **change) == code


@pytest.mark.parametrize("change, code", [
    ({"q": None}, 1), ({"out": None}, 1), ({"starts": None}, 1), ({"heads": 3}, 1), ({"heads": 0}, 1), ({"tokens": -1}, 1),
    ({"max_q": -1}, 1), ({"max_len": -1}, 1), ({"scale": -0.5}, 1), ({"scale": float("nan")}, 1),
    ({"scale": float("inf")}, 1), ({"sq": strides(252, 64)}, 3), ({"so": strides(256, -64)}, 3), ({"out": vp(0x1008)}, 3),
    ({"tokens": 1 << 30}, 3)])
def test_paged_attention_refuses(lib, change, code):
    assert attend(lib, **change) == code
    assert lib.sam_hip_last_error()


def test_launches_past_32_bits_of_threads_are_refused(lib):
    assert write(lib, tokens=1 << 26) == 3 and read(lib, max_len=1 << 25, batch=4) == 3
    size = lib.sam_hip_paged_attention_workspace_size
    # partial results that the joining launch has no threads for: no splits
    assert size(1, 1, 1 << 26, 1, 2, 2, 128, 1, 1 << 20) == 0 < size(1, 1, 1 << 20, 1, 2, 2, 128, 1, 1 << 20)


def test_a_token_that_no_launch_holds_is_refused(lib):
    """Threads of one token past what a launch counts: the host would have gone on without a token done."""
    for d in ((1 << 31) - 1, (1 << 31) - 255):
        assert rope(lib, b=1, l=1, h=1, d=d, pairs=0) == 3


def test_rows_whose_last_tile_passes_32_bits_are_refused(lib):
    size = lib.sam_hip_paged_attention_workspace_size
    for tokens in ((1 << 31) - 1, (1 << 31) - 255):
        assert attend(lib, tokens=tokens, heads=1, kv_heads=1, batch=1, max_q=1) == 3
        assert size(1, 1, tokens, 1, 1, 1, 64, 1, 64) == -1
    assert size(1, 1, (1 << 31) - 256, 1, 1, 1, 64, 1, 64) >= 0


def test_outputs_whose_rows_share_memory_are_refused(lib):
    assert attend(lib, so=strides(0, 64)) == 1 and attend(lib, so=strides(256, 0)) == 1
    assert rope(lib, so=strides(512, 0, 64)) == 1 and rope(lib, so=strides(512, 128, 0)) == 1
    assert rope(lib, b=2, so=strides(0, 128, 64)) == 1


def test_outputs_whose_rows_overlap_are_refused(lib):
    """Rows that share a part, by one stride or by two together; layouts whose rows lie apart get past that (to the
    refusal of an in-place call with other strides)."""
    for so in ((32, 64), (256, 56), (64, 64), (248, 64), (64, 192)):
        assert attend(lib, so=strides(*so)) == 1 and b"apart" in lib.sam_hip_last_error()
    for so in ((64, 256), (1 << 40, 64), (64, 1 << 60)):
        assert attend(lib, so=strides(*so)) == 1 and b"in place" in lib.sam_hip_last_error()
    for so in ((0, 64, 64), (0, 128, 32), (0, 120, 64), (512, 64, 64), (256, 128, 64)):
        assert rope(lib, b=2 if so[0] else 1, so=strides(*so)) == 1 and b"apart" in lib.sam_hip_last_error()
    for so in ((0, 64, 256), (0, 192, 64), (1 << 60, 64, 256), (8 * 64, 64, 4 * 64)):
        assert rope(lib, out=FAKE, b=2 if so[0] else 1, so=strides(*so)) == 1 and b"in place" in lib.sam_hip_last_error()


def test_attention_in_place_keeps_its_strides(lib):
    assert attend(lib, so=strides(512, 64)) == 1 and b"in place" in lib.sam_hip_last_error()
    assert attend(lib, sq=strides(64, 256), so=strides(256, 64)) == 1 and b"in place" in lib.sam_hip_last_error()
    need = dict(ws=None, d=128, kv_heads=1, batch=1, max_q=1, max_len=1 << 16, width=1 << 12)  # fails at its workspace
    assert attend(lib, tokens=1, heads=8, so=strides(1 << 20, 128), **need) == 1  # one token: its stride means nothing
    assert b"workspace" in lib.sam_hip_last_error()


def test_a_missing_or_short_workspace_is_refused(lib):
    size = lib.sam_hip_paged_attention_workspace_size
    need = size(1, 1, 1, 1, 8, 1, 128, 1, 1 << 16)
    assert need > 0 and size(1, 2, 1, 1, 8, 1, 128, 1, 64) == -1 and size(1, 1, 1, 1, 7, 2, 128, 1, 64) == -1
    big = dict(tokens=1, heads=8, kv_heads=1, d=128, batch=1, max_q=1, max_len=1 << 16, width=1 << 12)
    assert attend(lib, ws=None, ws_bytes=need, **big) == 1
    assert attend(lib, ws=FAKE, ws_bytes=need - 1, **big) == 1
    assert attend(lib, ws=vp(0x1008), ws_bytes=need, **big) == 3


def test_the_header_declares_what_the_library_exports(lib):
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "sam_hip_paged.h")).read()
    names = set(re.findall(r"\b(sam_hip_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == {"sam_hip_rope_axes", "sam_hip_kv_write", "sam_hip_kv_read", "sam_hip_paged_attention",
                     "sam_hip_paged_attention_workspace_size"}
    assert all(hasattr(lib, n) for n in names)


def test_the_switch_covers_the_paged_memory(lib):
    lib.sam_hip_set_enabled(0)
    try:
        assert rope(lib, x=None) == write(lib, k=None) == read(lib, k=None) == attend(lib, q=None) == 5
    finally:
        lib.sam_hip_set_enabled(1)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 64, dtype=torch.float16)
    pages, table = torch.zeros(4, 3, 16, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    one, two = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    freqs, axes = sam_hip.rope_freqs((16, 16), device="cpu")
    for call in (lambda: sam_hip.rope_axes(x, torch.zeros(2, 2, dtype=torch.int32), freqs, axes),
                 lambda: sam_hip.kv_write(x, x, pages, pages, table, two, one),
                 lambda: sam_hip.kv_read(pages, pages, table, one, 4),
                 lambda: sam_hip.paged_attention(x, pages, pages, table, two, one)):
        with pytest.raises(sam_hip.SamHipError, match="device tensors"):
            call()


def test_rope_freqs_are_the_axial_tables():
    freqs, axes = sam_hip.rope_freqs((64, 64), 10000.0, device="cpu")
    want = [10000.0 ** (-2 * j / 128) for j in range(64)]  # inv_j = theta^(-2j / (hd / 2)) at hd 256, vision.rs:26-46
    assert axes.tolist() == [0] * 64 + [1] * 64
    assert torch.allclose(freqs, torch.tensor(want + want, dtype=torch.float64), rtol=1e-14)
    with pytest.raises(sam_hip.SamHipError):
        sam_hip.rope_freqs((4, -1), device="cpu")


def test_reference_quantiser_rounds_to_the_nearest_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    grid = torch.unique(codes[torch.isfinite(codes)])
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 40, generator=g, dtype=torch.float64) * torch.pow(10.0, torch.randint(-3, 4, (64, 1), generator=g).double())
    x[0] = 0.0
    x[1, 0], x[2, 3] = float("inf"), float("nan")
    val, s = ref.quantise(x)
    for r in range(64):
        two = 2.0 ** (int(s[r]) - 127)
        fin = torch.isfinite(x[r])
        top = float(x[r][fin].abs().max())
        assert top <= 448 * two and (top == 0 or top > 224 * two)
        near = (x[r][fin][:, None] / two - grid).abs().min(-1).values
        assert torch.equal((val[r][fin] / two - x[r][fin] / two).abs(), near)
        assert torch.isnan(val[r][~fin]).all()
