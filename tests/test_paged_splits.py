"""Key splits of f32 attention over e2m1 pages: those of f32 pages, as the products bound both (CPU: the plan's workspace)."""
import os

import pytest

import sam_hip

F32, F16, E2M1 = 0, 1, 4


@pytest.fixture(scope="module")
def size():
    if not os.path.exists(sam_hip.LIB_PATH):
        pytest.skip("libsam_hip.so is not built")
    return sam_hip.load().sam_hip_paged_attention_workspace_size


@pytest.mark.parametrize("chunk, batch, group", [(1, 1, 1), (1, 1, 8), (1, 32, 4), (1, 64, 3), (4, 5, 2), (125, 9, 1), (125, 41, 1), (500, 1, 1), (2048, 1, 1)])
@pytest.mark.parametrize("heads, d", [(1, 96), (1, 128), (1, 256), (4, 64), (8, 128), (2, 32)])
@pytest.mark.parametrize("keys", [1, 577, 1024, 1500, 2048, 4320, 8192, 131072])
def test_f32_over_e2m1_is_split_as_over_f32(size, chunk, batch, group, heads, d, keys):
    call = (chunk * batch, batch, heads * group, heads, d, chunk, keys)
    assert size(F32, E2M1, *call) == size(F32, F32, *call) >= 0


def test_the_calls_that_the_rule_was_measured_at(size):
    """12 splits of 500 rows over 1500 keys, 8 of a token over 1024: partial results of d + 2 floats a row."""
    assert size(F32, E2M1, 500, 1, 1, 1, 128, 500, 1500) == 12 * 500 * 130 * 4
    assert size(F32, E2M1, 1, 1, 8, 8, 128, 1, 1024) == 8 * 8 * 130 * 4
    assert size(F16, E2M1, 1, 1, 8, 8, 128, 1, 1024) == 0  # 16 bits: conversions bound it, and a second launch costs more
