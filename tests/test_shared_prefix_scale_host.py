"""Shared-prefix decode refuses softmax scales that its tensor-core pass cannot take (no GPU needed)."""
from __future__ import annotations

import ctypes
import math

import pytest

from nvattn import _lib

FAKE = ctypes.c_void_p(0x10000)


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("batch,fp8", [(2, False), (2, True), (600, False), (600, True)])
def test_scale_is_refused_at_every_size(batch, fp8, scale):
    lib = _lib.load()
    scales = (FAKE, FAKE) if fp8 else (None, None)
    rc = lib.nvattn_shared_prefix_decode(
        FAKE, 1024, 128, FAKE, FAKE, *scales, FAKE, 1024, 128, FAKE, FAKE, 8, 8, 8, 128, 512, batch, 8, 2,
        128, ctypes.c_float(scale), FAKE, 1 << 40, None, None)
    assert rc == _lib.ERR_INVALID and b"softmax_scale" in lib.nvattn_last_error()
