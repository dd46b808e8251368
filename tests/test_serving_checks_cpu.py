"""Argument checks of the serving entry points' scale (no device is touched)."""
from __future__ import annotations

import ctypes
import math

import pytest

from test_serving_cpu import decode_args, lib, prompt_args  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("scale,code", [(0.125, 8), (2.3e38, 8), (3e38, 2), (math.inf, 2),
                                        (-math.inf, 2), (math.nan, 2), (-0.0, 2)])
def test_scale_has_to_be_positive_and_finite(lib, scale, code):  # noqa: F811
    assert lib.frsa_paged_decode(ctypes.byref(decode_args(lib, scale=scale)), None) == code
    assert lib.frsa_prompt_fwd(ctypes.byref(prompt_args(scale=scale)), None) == code
