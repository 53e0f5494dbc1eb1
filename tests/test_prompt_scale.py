"""CPU checks of the scales that whole prompts refuse."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    from heteroserve import _hip

    if not _hip.lib_path().exists():
        pytest.fail(f"{_hip.lib_path()} missing: run python hetero-serve_amd/build.py")
    return _hip.open_library()


@pytest.mark.parametrize("scale", [3.4e38, -3.4e38, 2.4e38, float("inf"), float("nan")])
def test_scales_whose_powers_of_2_are_not_finite(lib, scale):
    """The kernels work with scale times log2(e)."""
    one = ctypes.c_void_p(0x1000)
    rc = lib.hs_prompt_attention(one, one, one, 2, 256, 64, 128, 64, 128, 64, one, 1, 8, 8, 4, 2, 64,
                                 float(np.float32(scale)), one, None)
    assert rc == -1 and b"finite" in lib.hs_last_error()
