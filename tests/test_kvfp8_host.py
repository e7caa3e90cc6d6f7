"""fp8 KV cache, host side: the oracle's quantisation, and every refusal of the
C entry points and the operators (no GPU needed)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import reference_math as R

from nvattn import _lib, ops

FAKE = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10008)


def _err(rc, code, text):
    assert rc == code and text in _lib.load().nvattn_last_error().decode(), \
        (rc, _lib.load().nvattn_last_error())


def test_oracle_rows_keep_half_a_step():
    """|x8 2^k - x| <= 2^-4 |x| for normal e4m3 results, half of the subnormal
    step 2^-9 * 2^k below 2^-6 * 2^k; the scale is the smallest allowed."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(200, 128, generator=g) * torch.exp2(torch.randint(-30, 30, (200, 1),
                                                                      generator=g).float()))
    x = x.to(torch.bfloat16).double()
    q, e = R.quantise_rows_fp8(x)
    back = R.expand_rows_fp8(q, e)
    s = torch.exp2(e.double() - 127)[:, None]
    assert ((back - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10)).all()
    amax = x.abs().amax(-1)
    assert (amax <= 448 * s[:, 0]).all() and (amax > 224 * s[:, 0]).all()


def test_oracle_rows_edges():
    x = torch.zeros(6, 128)
    x[1, 5] = 448.0
    x[2, 5] = 450.0                       # bf16's next value above 448
    x[3, 5] = float("inf")
    x[4, 5] = float("nan")
    x[5, 5] = 2.0 ** -130
    q, e = R.quantise_rows_fp8(x.to(torch.bfloat16))
    assert e.tolist() == [27, 127, 128, 255, 255, 27]
    back = R.expand_rows_fp8(q, e)
    assert back[1, 5] == 448 and back[2, 5] == 448 and torch.isnan(back[3:5]).all()
    assert (back[0] == 0).all() and (back[5] == 0).all()


def _store(n=4, kvh=2, hd=128, nb=8, bs=64, key=FAKE, kc=FAKE, ks=FAKE, stride=512):
    return _lib.load().nvattn_store_kvcache_fp8(key, stride, FAKE, stride, kc, FAKE, ks, FAKE,
                                                FAKE, n, kvh, hd, nb, bs, None, None)


def test_store_refusals():
    assert _store(n=0, key=None) == _lib.OK
    _err(_store(n=-1), _lib.ERR_INVALID, "negative")
    _err(_store(key=None), _lib.ERR_INVALID, "NULL")
    _err(_store(ks=None), _lib.ERR_INVALID, "NULL")
    _err(_store(hd=64), _lib.ERR_UNSUPPORTED, "head_dim")
    _err(_store(nb=0), _lib.ERR_INVALID, "geometry")
    _err(_store(stride=255), _lib.ERR_INVALID, "overlap")
    _err(_store(kc=ODD), _lib.ERR_INVALID, "16-byte")
    _err(_store(key=ctypes.c_void_p(0x10001)), _lib.ERR_INVALID, "2-byte")


def _load(s=2, total=10, hd=128, bs=64, kc=FAKE, ko=FAKE, stride=4, width=4):
    return _lib.load().nvattn_load_kvcache_fp8(kc, FAKE, FAKE, FAKE, FAKE, s, FAKE, stride, width, 8,
                                               bs, 2, hd, total, 0, ko, FAKE, None, None)


def test_load_refusals():
    assert _load(s=0) == _lib.OK and _load(total=0, ko=None) == _lib.OK
    _err(_load(s=-1), _lib.ERR_INVALID, "negative")
    _err(_load(kc=None), _lib.ERR_INVALID, "NULL")
    _err(_load(hd=256), _lib.ERR_UNSUPPORTED, "head_dim")
    _err(_load(bs=0), _lib.ERR_INVALID, "geometry")
    _err(_load(stride=3), _lib.ERR_INVALID, "geometry")
    _err(_load(ko=ODD), _lib.ERR_INVALID, "16-byte")


def _decode(batch=2, heads=8, kvh=2, hd=128, bs=64, width=64, ks=FAKE, ws=None, wsb=0, q=FAKE,
            stride=64):
    return _lib.load().nvattn_paged_decode_fp8(
        q, heads * hd, hd, FAKE, FAKE, ks, FAKE, FAKE, heads * hd, hd, FAKE, FAKE, stride, width, 8,
        bs, batch, heads, kvh, hd, ctypes.c_float(0.1), ws, wsb, None, None)


def test_decode_refusals():
    assert _decode(batch=0, q=None) == _lib.OK
    _err(_decode(batch=-1), _lib.ERR_INVALID, "paged_decode_fp8: negative batch")
    _err(_decode(q=None), _lib.ERR_INVALID, "NULL")
    _err(_decode(ks=None), _lib.ERR_INVALID, "NULL scales")
    _err(_decode(ks=ODD), _lib.ERR_INVALID, "scales must be 16-byte")
    _err(_decode(hd=64), _lib.ERR_UNSUPPORTED, "head_dim")
    _err(_decode(heads=9), _lib.ERR_INVALID, "multiple of num_kv_heads")
    _err(_decode(heads=64), _lib.ERR_UNSUPPORTED, "16 query heads")
    _err(_decode(bs=96), _lib.ERR_UNSUPPORTED, "multiple of 64")
    _err(_decode(stride=63), _lib.ERR_INVALID, "geometry")
    _err(_decode(batch=70000), _lib.ERR_UNSUPPORTED, "65535")
    _err(_decode(width=(1 << 24) + 1, stride=1 << 25), _lib.ERR_UNSUPPORTED, "2^30 keys")
    _err(_decode(), _lib.ERR_WORKSPACE, "workspace")
    _err(_decode(ws=ctypes.c_void_p(0x10010), wsb=1 << 30), _lib.ERR_INVALID, "256-byte")


def test_operators_refuse_cpu_tensors_and_wrong_types():
    kc = torch.zeros(2, 64, 2, 128, dtype=torch.float8_e4m3fn)
    ks = torch.zeros(2, 2, 64, dtype=torch.uint8)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.store_kvcache_fp8(x, x, kc, kc, ks, ks, i32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.load_kvcache_fp8(kc, kc, ks, ks, i32, i32.view(3, 1), 3)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_fp8(x, kc, kc, ks, ks, i32, i32.view(3, 1))
    # the shape checks themselves, which run before any launch
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops._check_fp8_caches(kc.view(torch.uint8), kc, ks, ks)
    with pytest.raises(TypeError, match="uint8"):
        ops._check_fp8_caches(kc, kc, ks.float(), ks)
    with pytest.raises(ValueError, match="k_scale"):
        ops._check_fp8_caches(kc, kc, ks.transpose(1, 2).contiguous(), ks)
    with pytest.raises(ValueError, match="contiguous"):
        ops._check_fp8_caches(kc[:, :, :, :].transpose(1, 2).contiguous().transpose(1, 2), kc, ks, ks)
    with pytest.raises(ValueError, match="one row"):
        ops._check_table(i32.view(3, 1), 2)
    with pytest.raises(TypeError, match="int32"):
        ops._check_table(i32.view(3, 1).long(), 3)
    assert np.array_equal(kc.shape, (2, 64, 2, 128))


def test_module_needs_the_exponents_of_an_fp8_cache():
    import nvattn
    attn = nvattn.Attention(4, 128, 0.1, 2)
    attn.k_cache = attn.v_cache = torch.zeros(2, 64, 2, 128, dtype=torch.float8_e4m3fn)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k_scale"):
        attn(x, x, x)
