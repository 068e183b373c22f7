"""The spectral caches' calls refuse rows of a type that they do not have, bf16 among them (the 8-bit
block cache's alone), before they look at anything else."""
import ctypes as C

import pytest

import sp_hip as S

# entry point -> its arguments but for the type, which stands where None does
BATCH = (None, 0, 0, 0, 0, 4, 4096)  # cache, is_v, layer, head, start, n, rows
LAYER = (None, 0, 0, 4, 4096, 4096, 512)
ALL = (None, 0, 4, 4096, 4096)
ENCODE = (None, None, 0, 4096)
CALLS = {
    "sp_hip_write_layer": (LAYER, ()),
    "sp_hip_read_layer": (LAYER, (-1,)),
    "sp_hip_write_all": (ALL, ()),
    "sp_hip_read_all": (ALL, (-1,)),
    "sp_hip_sqfree_write_batch": (BATCH, ()),
    "sp_hip_sqfree_read_batch": (BATCH, ()),
    "sp_hip_sqfree_write_layer": (LAYER, ()),
    "sp_hip_sqfree_read_layer": (LAYER, ()),
    "sp_hip_hier_write_batch": (BATCH, ()),
    "sp_hip_hier_read_batch": (BATCH, ()),
    "sp_hip_hier_write_layer": (LAYER, ()),
    "sp_hip_hier_read_layer": (LAYER, ()),
    "sp_hip_ship_encode": (ENCODE, (0, 128, 4096, 0, 1, 4, None)),
    "sp_hip_ship_encode_generic": (ENCODE, (0, 128, 4096, 0, 1, 4, None)),
    "sp_hip_ship_decode": ((None, None, 0, -1, 4096, 0, 4096), (0, 128, 1, 4, None)),
    "sp_hip_ship_decode_generic": ((None, None, 0, -1, 4096, 0, 4096), (0, 128, 1, 4, None)),
}


@pytest.mark.parametrize("dtype", [S.DTYPE_BF16, 3, -1])
@pytest.mark.parametrize("name", list(CALLS))
def test_unknown_row_types_are_refused(name, dtype):
    before, after = CALLS[name]
    assert getattr(S.lib(), name)(*before, dtype, *after) == -1
    assert f"dtype {dtype}" in S.last_error()


@pytest.mark.parametrize("name,args", [
    ("sp_hip_roundtrip_cells", (None, 0, 4096, 1, 4096, 512, 4096, 512, 1, S.DTYPE_BF16, -1, None)),
    ("sp_hip_calibrate_feed", (None, 4096, 128, 4, S.DTYPE_BF16)),
    ("sp_hip_sqfree_calibrate_feed", (None, 4096, 128, 4, S.DTYPE_BF16)),
    ("sp_hip_hier_calibrate_feed", (None, 0, 4096, 128, 4, S.DTYPE_BF16)),
    ("sp_hip_dual_write_layer", (None, 0, 0, 4, 4096, 4096, 512, S.DTYPE_BF16)),
    ("sp_hip_dual_read_merged", (None, 0, 4, 4096, 4096, 512, S.DTYPE_BF16)),
])
def test_calls_that_asked_before_still_do(name, args):
    assert getattr(S.lib(), name)(*args) == -1
    assert S.last_error().endswith("bad args")


def test_every_call_with_a_row_type_is_here():
    """Every function of the header whose last arguments name a dtype, but for the block cache's."""
    import os
    import re
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(S.INCLUDE_DIR, "sp_hip.h")).read(), flags=re.S)
    named = {m.group(1) for m in re.finditer(r"(sp_hip_\w+)\s*\(([^;]*?)\)\s*;", text) if "dtype" in m.group(2)}
    asked = {"sp_hip_roundtrip_cells", "sp_hip_calibrate_feed", "sp_hip_sqfree_calibrate_feed",
             "sp_hip_hier_calibrate_feed", "sp_hip_dual_write_layer", "sp_hip_dual_read_merged"}
    assert {n for n in named if not n.startswith("sp_hip_fp8_")} == set(CALLS) | asked
