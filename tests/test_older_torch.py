"""A torch without the 4-bit type has every operator but the 4-bit ones, whose refusal says why (CPU only)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys
import torch

del torch.float4_e2m1fn_x2
sys.path.insert(0, sys.argv[1])
import sam_encoder
import sam_hip

assert not hasattr(torch, "float4_e2m1fn_x2")
sam_hip._device_of = lambda what, *ts: 0
sam_hip._is_current = lambda dev: True


def refused(call, words):
    try:
        call()
    except sam_hip.SamHipError as e:
        assert words in str(e), e
    else:
        raise AssertionError("no refusal")


dt = sam_hip._dtype
sam_hip._dtype = lambda *ts: sam_hip._DTYPES[ts[0].dtype]
x, codes, scale = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
for call in (lambda: sam_hip.mx_pack(x), lambda: sam_hip.mx_unpack(codes, scale), lambda: sam_hip.mx_matmul(codes, scale, codes, scale),
             lambda: sam_hip.mx_linear(x, codes, scale)):
    refused(call, "float4_e2m1fn_x2")
sam_hip._dtype = dt

# a pool of 16 or 8 bits is taken as it was
i = lambda *a: torch.zeros(a, dtype=torch.int32)
pages, byte = torch.zeros(4, 3, 16, 64, dtype=torch.float16), torch.zeros(4, 3, 16, dtype=torch.uint8)
args = i(1, 2), i(2), i(1), torch.float16
assert sam_hip._pool("call", pages, pages, None, None, *args)[0] == 1
assert sam_hip._pool("call", pages.to(torch.float8_e4m3fn), pages.to(torch.float8_e4m3fn), byte, byte, *args)[0] == 3
refused(lambda: sam_hip._pool("call", pages.to(torch.uint8), pages.to(torch.uint8), byte, byte, *args), "the cache must hold")
print("done")
"""


def test_import_and_refusals_without_the_type():
    if not os.path.exists(os.path.join(ROOT, "sam-rs_amd", "libsam_hip.so")):
        pytest.skip("libsam_hip.so is not built")
    r = subprocess.run([sys.executable, "-c", PROGRAM, os.path.join(ROOT, "sam-rs_amd")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr
