"""Prefix-cache prefill through the module with a sequence longer than its table: flagged, over an fp8
cache as over a bf16 one."""
from __future__ import annotations

import pytest
import torch

from helpers import cu

import nvattn
from nvattn import context as ctxmod
from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tot", [[256], [257], [400], [256, 100], [100, 257], [60, 500, 256]])
def test_lengths_past_the_table(tot, fp8):
    bs, kvh, add = 128, 2, [5] * len(tot)
    attn = nvattn.Attention(4, 128, 128 ** -0.5, kvh)
    attn.k_cache, attn.v_cache = [torch.zeros(6, bs, kvh, 128, dtype=torch.bfloat16, device=dev) for _ in "kv"]
    if fp8:
        attn.k_cache, attn.v_cache = [c.to(torch.float8_e4m3fn) for c in (attn.k_cache, attn.v_cache)]
        attn.k_scale, attn.v_scale = [torch.full((6, kvh, bs), 127, dtype=torch.uint8, device=dev) for _ in "kv"]
    bt = torch.arange(2 * len(tot), dtype=torch.int32, device=dev).view(-1, 2)
    n = sum(add)
    q, k, v = [torch.zeros(n, h, 128, dtype=torch.bfloat16, device=dev) for h in (4, kvh, kvh)]
    skip = torch.full((n,), -1, dtype=torch.int32, device=dev)
    ctxmod.set_context(True, cu(add).to(dev), cu(tot).to(dev), max(add), max(tot), skip, None, bt)
    ops.read_status()
    attn(q, k, v)
    ctxmod.reset_context()
    assert ops.read_status() == (nvattn._lib.STATUS_BAD_BLOCK if max(tot) > 2 * bs else 0)
