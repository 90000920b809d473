"""sam_hip_kv_append refuses bad arguments before touching a GPU (CPU only: no kernel is launched)."""
import ctypes
import os
import re

import pytest
import torch

import sam_hip
from test_paged_abi import BAD_POOL, FAKE, POOL, strides

vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    return sam_hip.load()


def append(lib, q=FAKE, k=FAKE, v=FAKE, pos=FAKE, freqs=FAKE, axes=FAKE, out=vp(0x2000), starts=FAKE, tokens=4, heads=4, pairs=16, naxes=2,
           sq=None, sk=None, sv=None, sp=None, so=None, **change):
    a = {**POOL, **change}
    return lib.sam_hip_kv_append(q, k, v, pos, freqs, axes, out, a["k_pages"], a["v_pages"], a["ks"], a["vs"], a["table"], starts, a["lens"],
                                 a["dtype"], a["cache"], tokens, a["batch"], heads, a["pages"], a["kv_heads"], a["page"], a["d"], a["width"],
                                 pairs, naxes, sq, sk, sv, sp, so, 0, 0, None)


@pytest.mark.parametrize("change, code", BAD_POOL + [({"cache": 4, "d": 72}, 3), ({"cache": 4, "vs": None}, 1), ({"cache": 5}, 2)])
def test_bad_pools_are_refused(lib, change, code):
    assert append(lib, **change) == code
    assert lib.sam_hip_last_error()


@pytest.mark.parametrize("change, code", [
    ({"k": None}, 1), ({"v": None}, 1), ({"starts": None}, 1), ({"q": None}, 1), ({"out": None}, 1), ({"freqs": None}, 1), ({"axes": None}, 1),
    ({"tokens": -1}, 1), ({"heads": 0}, 1), ({"pairs": -1}, 1), ({"pairs": 33}, 1), ({"naxes": 0}, 1), ({"tokens": 1 << 26}, 3),
    ({"tokens": (1 << 26) - 8, "heads": 1, "kv_heads": 1}, 3), ({"heads": 65536}, 3), ({"sq": strides(252, 64)}, 3), ({"sk": strides(100, 64)}, 3), ({"sv": strides(-128, 64)}, 3),
    ({"so": strides(256, -64)}, 3), ({"so": strides(64, 64)}, 1), ({"sp": strides(-2, 1)}, 3), ({"q": vp(0x1008)}, 3), ({"k": vp(0x1002)}, 3),
    ({"out": vp(0x2008)}, 3), ({"pos": vp(0x1002)}, 3), ({"freqs": vp(0x1004)}, 3), ({"axes": vp(0x1001)}, 3),
    ({"out": FAKE, "sq": strides(512, 64)}, 1)])
def test_bad_arguments_are_refused(lib, change, code):
    assert append(lib, **change) == code
    assert lib.sam_hip_last_error()


def test_calls_without_work_and_the_switch(lib):
    assert append(lib, tokens=0) == 0 and append(lib, tokens=0, q=None, out=None, heads=0) == 0
    assert append(lib, tokens=0, pairs=0, pos=None, freqs=None, axes=None) == 0 and append(lib, tokens=0, pos=None, axes=None, naxes=0) == 0
    lib.sam_hip_set_enabled(0)
    try:
        assert append(lib, k=None) == 5
    finally:
        lib.sam_hip_set_enabled(1)


def test_the_header_declares_what_the_library_exports(lib):
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "sam_hip_append.h")).read()
    names = set(re.findall(r"\b(sam_hip_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == {"sam_hip_kv_append"} and hasattr(lib, "sam_hip_kv_append")


def test_cpu_tensors_are_refused():
    x, pages = torch.zeros(2, 3, 64, dtype=torch.float16), torch.zeros(4, 3, 16, 64, dtype=torch.float16)
    one, two, table = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    freqs, axes = sam_hip.rope_freqs((16,), device="cpu")
    with pytest.raises(sam_hip.SamHipError, match="device tensors"):
        sam_hip.kv_append(x, x, x, freqs, axes, pages, pages, table, two, one)
