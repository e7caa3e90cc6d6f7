"""Prefill of a batch in which one sequence's keys and values are not finite: the others' outputs are bit
for bit what they are without it, also where a key tile reaches into the neighbour's rows."""
from __future__ import annotations

import pytest
import torch

from helpers import cu

import nvattn
from nvattn import context as ctxmod
from nvattn import ops
from oracle import reference_math as R

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
SCALE = 128 ** -0.5
H, KVH = 8, 2


def _rows(cu_q, seqs):
    return torch.cat([torch.arange(int(cu_q[b]), int(cu_q[b + 1])) for b in seqs])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,new", [([100, 130, 64], [100, 130, 64]), ([129, 1, 300, 256], [1, 1, 300, 7]),
                                      ([383, 40, 20], [250, 40, 3])])
def test_dense(lens, new, causal, bad):
    g = torch.Generator().manual_seed(sum(lens))
    q = torch.randn(sum(new), H, 128, generator=g).to(torch.bfloat16).to(dev)
    k, v = [torch.randn(sum(lens), KVH, 128, generator=g).to(torch.bfloat16).to(dev) for _ in "kv"]
    cq, ck = cu(new), cu(lens)

    def run(k, v):
        return ops.varlen_prefill(q, k, v, cq.to(dev), ck.to(dev), max(new), max(lens), SCALE, causal)
    clean = run(k, v)
    assert torch.isfinite(clean.float()).all()
    for b in range(len(lens)):
        kb, vb = k.clone(), v.clone()
        kb[ck[b]:ck[b + 1]] = bad
        vb[ck[b]:ck[b + 1]] = bad
        at = _rows(cq, [i for i in range(len(lens)) if i != b]).to(dev)
        assert torch.equal(run(kb, vb)[at], clean[at]), b


def test_prefix_cache_over_an_fp8_cache():
    """The same through the module: a sequence whose stored rows are NaN beside two whose are not."""
    bs, tot, add = 64, [300, 100, 130], [7, 100, 33]
    g = torch.Generator().manual_seed(7)
    bt = torch.arange(15, dtype=torch.int32).view(3, 5)
    cq, ck = cu(add), cu(tot)
    q, k, v = [torch.randn(sum(add), h, 128, generator=g).to(torch.bfloat16).to(dev) for h in (H, KVH, KVH)]
    attn = nvattn.Attention(H, 128, SCALE, KVH)
    start = [R.quantise_rows_fp8(torch.randn(15, bs, KVH, 128, generator=g).to(torch.bfloat16)) for _ in "kv"]
    skip = torch.full((sum(add),), -1, dtype=torch.int32, device=dev)

    def run(bad=None):
        for name, (c, e) in zip("kv", start):
            c, e = c.clone(), e.transpose(1, 2).contiguous()
            if bad is not None:
                c.view(torch.uint8)[bt[bad].long()] = 0x7F
                e[bt[bad].long()] = 255
            setattr(attn, f"{name}_cache", c.to(dev))
            setattr(attn, f"{name}_scale", e.to(dev))
        ctxmod.set_context(True, cq.to(dev), ck.to(dev), max(add), max(tot), skip, None, bt.to(dev))
        o = attn(q, k, v)
        ctxmod.reset_context()
        return o
    clean = run()
    assert torch.isfinite(clean.float()).all()
    for b in range(3):
        at = _rows(cq, [i for i in range(3) if i != b]).to(dev)
        o = run(b)
        assert torch.equal(o[at], clean[at]), b
        assert torch.isnan(o[_rows(cq, [b]).to(dev)].float()).all()
