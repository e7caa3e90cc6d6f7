"""Rows whose scores lie hundreds of powers of two apart, in every tensor-core attention mode: weights far
below the row's largest are zeros, whichever unit takes their exponential."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import cu, paged_layout
from oracle import reference_math as R

from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
SCALE = 128 ** -0.5
H, KVH, BS = 8, 2, 128


def _keys(shape, g):
    """Normal keys of which random ones are 20 times as large: their scores are +-30 (in powers of two)
    and more, next to others near zero, within every tile."""
    k = torch.randn(shape, generator=g)
    return torch.where(torch.rand(*shape[:-1], 1, generator=g) < 0.3, 20 * k, k).to(torch.bfloat16)


def _check(out, ref, mix, q, k, what):
    """|out - ref| element by element, against the arithmetic: the output is rounded to bf16, 2^-8 of
    it; the weights p_j go to the tensor cores as bf16, 2^-8 each, and take exp2 from a polynomial,
    7.5e-5 in the weight and in the sum, so that much of mix = sum_j p_j |v_j|; a score sums 128
    products in fp32, off by 136 * 2^-24 of sum |q_d k_d| <= |q| |k| in the kernel and in the fp32
    oracle, in the weight and in the sum. (These rows are mixes of one or two V rows of up to 4: the
    weights' rounding alone is 2^-8 * 4.)"""
    dot = (q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max() * SCALE).item()
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 1.5e-4 + 4 * 136 * 2.0 ** -24 * dot) * mix
    err = (out.float().cpu() - ref.float()).abs()
    print(f"[max-abs] score spread, {what}: {err.max():.3e}, margin {(tol - err).min():.3e}")
    assert not torch.isnan(out).any() and (err <= tol).all()


def _cache(lens, seed):
    g = torch.Generator().manual_seed(seed)
    blocks, bt = paged_layout(lens, BS, seed=seed)
    k = _keys((blocks, BS, KVH, 128), g)
    v = torch.randn(blocks, BS, KVH, 128, generator=g).to(torch.bfloat16)
    return k, v, bt, g


@pytest.mark.parametrize("paged", [False, True])
def test_prefill(paged):
    lens, new = [512, 300, 900], [512, 100, 700]
    k, v, bt, g = _cache(lens, 1)
    q = torch.randn(sum(new), H, 128, generator=g).to(torch.bfloat16)
    cq, ck = cu(new), cu(lens)
    kd, vd = [torch.cat([R.gather_paged(c, bt[b].numpy(), n) for b, n in enumerate(lens)])
              .to(torch.bfloat16) for c in (k, v)]
    ref, mix = [R.varlen_attention(q, kd, x, cq.numpy(), ck.numpy(), SCALE, True) for x in (vd, vd.abs())]
    kv = (k, v) if paged else (kd, vd)
    out = ops.varlen_prefill(q.to(dev), *(t.to(dev) for t in kv), cq.to(dev), ck.to(dev), max(new),
                             max(lens), SCALE, True, bt.to(dev) if paged else None)
    _check(out, ref, mix, q, k, f"{'paged' if paged else 'dense'} prefill")


def test_tree():
    n = 16
    ctx = [500, 130, 1000]
    k, v, bt, g = _cache([c + n for c in ctx], 2)
    q = torch.randn(n * len(ctx), H, 128, generator=g).to(torch.bfloat16)
    mask = torch.tensor([(2 << j) - 1 for j in range(n)] * len(ctx), dtype=torch.int64)  # chains
    cq, lens = cu([n] * len(ctx)), torch.tensor(ctx, dtype=torch.int32)
    ref, mix = [R.tree_attention(q, k, x, cq.numpy(), lens.numpy(), mask.numpy(), bt.numpy(), SCALE)
                for x in (v, v.abs())]
    out = ops.tree_attention(q.to(dev), k.to(dev), v.to(dev), cq.to(dev), lens.to(dev), mask.to(dev),
                             bt.to(dev), n, SCALE)
    _check(out, ref, mix, q, k, "tree")


def test_shared_prefix():
    shared, B = 1024, 80
    k, v, bt, g = _cache([shared] + [100] * B, 3)
    table = torch.cat([bt[:1, :shared // BS].expand(B, -1), bt[1:, :1]], 1).contiguous()
    lens = np.full(B, shared + 100)
    q = torch.randn(B, H, 128, generator=g).to(torch.bfloat16)
    ref, mag = R.decode_attention_f64(q, k.double(), v.double(), lens, table, SCALE)
    out = ops.shared_prefix_decode(q.to(dev), k.to(dev), v.to(dev),
                                   torch.from_numpy(lens).int().to(dev), table.to(dev), shared, SCALE)
    _check(out, ref, mag["mix"], q, k, "shared prefix")
