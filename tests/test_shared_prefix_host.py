"""Shared-prefix decode, host side: refusals of the C entry point and the operator,
and what its split policy makes of host sizes (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from nvattn import _lib, ops

FAKE = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10008)


def _call(batch=2, heads=8, kvh=2, hd=128, bs=128, width=4, shared=128, q=FAKE, ks=None, vs=None,
          ws=FAKE, wsb=1 << 40, qstride=1024):
    return _lib.load().nvattn_shared_prefix_decode(
        q, qstride, hd, FAKE, FAKE, ks, vs, FAKE, heads * hd, hd, FAKE, FAKE, width, width, 8, bs,
        shared, batch, heads, kvh, hd, ctypes.c_float(0.1), ws, wsb, None, None)


def test_c_refusals():
    lib = _lib.load()
    assert _call(batch=0, q=None) == _lib.OK
    for kw, code, text in ((dict(batch=-1), _lib.ERR_INVALID, b"negative batch"),
                           (dict(q=None), _lib.ERR_INVALID, b"NULL"),
                           (dict(hd=64), _lib.ERR_UNSUPPORTED, b"head_dim"),
                           (dict(heads=34, kvh=2), _lib.ERR_UNSUPPORTED, b"16 query heads"),
                           (dict(bs=64, shared=64), _lib.ERR_UNSUPPORTED, b"multiple of 128"),
                           (dict(shared=100), _lib.ERR_INVALID, b"whole blocks"),
                           (dict(shared=-128), _lib.ERR_INVALID, b"whole blocks"),
                           (dict(shared=5 * 128), _lib.ERR_INVALID, b"whole blocks"),
                           (dict(ks=FAKE), _lib.ERR_INVALID, b"NULL scales"),
                           (dict(ks=FAKE, vs=ODD), _lib.ERR_INVALID, b"scales must be"),
                           (dict(q=ODD), _lib.ERR_UNSUPPORTED, b"16-byte multiples"),
                           (dict(qstride=1020), _lib.ERR_UNSUPPORTED, b"16-byte multiples"),
                           (dict(batch=70000), _lib.ERR_UNSUPPORTED, b"65535"),
                           (dict(width=1 << 24), _lib.ERR_UNSUPPORTED, b"2^30 keys"),
                           (dict(ws=None), _lib.ERR_WORKSPACE, b"workspace"),
                           (dict(wsb=16), _lib.ERR_WORKSPACE, b"workspace"),
                           (dict(ws=ODD), _lib.ERR_INVALID, b"256-byte")):
        assert _call(**kw) == code and text in lib.nvattn_last_error(), (kw, lib.nvattn_last_error())


def test_workspace_depends_on_host_sizes():
    f = ops.shared_prefix_workspace_bytes
    slot = 128 * 4 + 8
    # nothing shared: the own keys' partials, one split at least
    assert f(4, 8, 2, 1, 128, 0) >= 4 * 8 * slot
    # an fp8 prefix that is attended apart adds its bf16 rows
    assert f(200, 8, 2, 9, 128, 1024, True) - f(200, 8, 2, 9, 128, 1024) == 2 * 1024 * 2 * 128 * 2
    # a short one of few rows is read with the own keys: no partials of its own
    assert f(4, 8, 2, 9, 128, 1024) < f(100, 8, 2, 9, 128, 1024) // 25
    # sizes that the call refuses need no workspace
    assert f(4, 8, 2, 9, 128, 100) == 0 and f(0, 8, 2, 9, 128, 128) == 0
    assert f(4, 8, 3, 9, 128, 128) == 0 and f(4, 8, 2, 9, 128, 10 * 128) == 0


def test_operator_refuses_cpu_tensors():
    q = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    c = torch.zeros(1, 128, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_prefix_decode(q, c, c, i, i.view(1, 1), 128)
